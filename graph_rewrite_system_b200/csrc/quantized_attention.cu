// One query per sequence against 8-bit pages: grs_quantized_attention.
//
// softmax(scale q k) v with k and v an e4m3 code times the scale of its page and
// head.  e4m3 is exact in f16, so the codes go into f16 tensor-core products as
// they are and the scales join in fp32: the key scale multiplies the score, the
// value scale's log2 is added to it before the exponential that weighs the values.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "e4m3.cuh"

namespace grs {

struct QuantArgs {
  const void* q; int64_t q_sb, q_sh;
  const uint8_t* kc; const uint8_t* vc; int64_t c_sp, c_st, c_sh;
  const float* ks; const float* vs; int64_t s_sp;
  const int32_t* bt; int64_t bt_s; int columns; const int32_t* lengths; int pages, page;
  bool q_whole;                             // query rows in 16-byte pieces
  uint32_t magic; int shift;                // t / page = umulhi(t, magic) >> shift; magic 0: page 1
  float* part; float* part_lse; int slices;             // partial sums
  int ranges; int32_t* starts;              // of the stream form; first tiles of the sequences
  bool o_whole;                             // output rows in pieces of four elements
  void* out; int64_t o_sb, o_sh;
  int batch, heads, kv_heads, group, D;
  float scale_log2;
  int32_t* status;
};

constexpr float QA_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ int quant_length(const QuantArgs& a, int b, bool by_warp = false) {
  const bool tells = (threadIdx.x & (by_warp ? 31 : ~0)) == 0;
  const int room = a.columns * a.page, length = __ldg(a.lengths + b);
  const int past = min(max(length, 0), room);
  if (past != length && tells) set_status(a.status, GRS_ERR_LENGTH);
  if (a.pages == 0 && past > 0) {           // no address to read from
    if (tells) set_status(a.status, GRS_ERR_BAD_PAGE);
    return 0;
  }
  return past;
}

// ---- any layout ---------------------------------------------------------------
// One CTA of four warps per sequence and query head, every warp taking each fourth
// run of 32 tokens: a lane per key for the scores, a lane per column for the
// values, byte loads.  For widths that are no multiple of 8 and rows off 8 bytes; bound
// by its loads, one code each.
template <typename T>
__global__ void __launch_bounds__(128) quant_rows_kernel(QuantArgs a) {
  constexpr int ND = 8;
  __shared__ float q[256], sums[4][256], tops[4], totals[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / a.heads, head = blockIdx.x % a.heads, h = head / a.group;
  const T* query = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)head * a.q_sh;
  for (int d = threadIdx.x; d < a.D; d += 128) q[d] = to_float(query[d]) * a.scale_log2;
  const int past = quant_length(a, b);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[ND] = {};
  for (int t0 = 32 * warp; t0 < past; t0 += 128) {
    const int t = t0 + lane;
    const uint8_t* v = nullptr;
    float s = -INFINITY, vs = 0.f;
    if (t < past) {
      const int page = __ldg(a.bt + (int64_t)b * a.bt_s + t / a.page);
      if (page < 0 || page >= a.pages) {
        set_status(a.status, GRS_ERR_BAD_PAGE);
      } else {
        const int64_t at = (int64_t)page * a.c_sp + (int64_t)(t % a.page) * a.c_st + h * a.c_sh;
        v = a.vc + at;
        vs = a.vs[page * a.s_sp + h];
        s = 0.f;
        for (int d = 0; d < a.D; ++d) s = fmaf(q[d], from_e4m3(a.kc[at + d]), s);
        s *= a.ks[page * a.s_sp + h];
      }
    }
    const float top = fmaxf(m, warp_max(s)), base = top == -INFINITY ? 0.f : top;
    const float p = exp2f(s - base), keep = exp2f(m - base);
    l = l * keep + p;
    m = top;
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] *= keep;
    for (int j = 0; j < 32; ++j) {
      const uint8_t* vj = reinterpret_cast<const uint8_t*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v), j));
      const float w = __shfl_sync(0xffffffffu, p * vs, j);
      if (!vj) continue;
#pragma unroll
      for (int i = 0; i < ND; ++i)
        if (lane + 32 * i < a.D) acc[i] = fmaf(w, from_e4m3(vj[lane + 32 * i]), acc[i]);
    }
  }
  l = warp_sum(l);
  if (lane == 0) tops[warp] = m, totals[warp] = l;
#pragma unroll
  for (int i = 0; i < ND; ++i) sums[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float base = top == -INFINITY ? 0.f : top;
  float w[4], norm = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = exp2f(tops[i] - base);
    norm += w[i] * totals[i];
  }
  const float inv = norm == 0.f ? 0.f : 1.f / norm;
  T* out = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)head * a.o_sh;
  for (int d = threadIdx.x; d < a.D; d += 128)
    out[d] = from_float<T>(((w[0] * sums[0][d] + w[1] * sums[1][d]) +
                            (w[2] * sums[2][d] + w[3] * sums[3][d])) * inv);
}

// ---- tensor cores ---------------------------------------------------------------
// A warp streams tiles of 16 tokens of one (sequence, K/V head) through a ring of
// its own in shared memory: cp.async fetches the rows in 16-byte pieces wherever
// their pages lie, two or three steps ahead.  Keys, then value columns, are the 16 rows of
// mma.m16n8k16, the group's query heads its columns.  The order in which a product
// sums its inner dimension is free, so a lane takes whole pieces of a row, and a
// lane's column index picks its piece of the value rows; two tokens' codes are
// interleaved by byte permutes before they are widened.  Lane i looks up one run of 8
// tokens for 16 tiles at once, and shuffles hand places and scales round (a look-up per
// token and tile: 79 us against 70 for 64 sequences of up to 4099 tokens).
constexpr int QT_WARPS = 4;
constexpr int QT_STAGES = 3;
// Weights go into the value products in f16: the largest between 2^9 and 2^15, the smallest
// that it holds 2^-24, 2^-33 of the largest.  One f16 is off by 2^-11 of a weight at most,
// 2e-4 in the mean, beside the 1.7e-3 of the norm that rounding the output to bf16 costs;
// fp32 takes two parts, 22 bits, for queries and weights.
constexpr float QT_LIFT = 9.f;
constexpr float QT_SLACK = 6.f;
constexpr uint32_t QT_ABSENT = 0xffffffffu; // key scale of a token that is not there
constexpr float QT_UNSET = -3e38f;          // a reference before the first score

__device__ __forceinline__ void qt_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void qt_widen(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ float qt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t qt_pack(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// x - its f16 value, for the second part of an fp32 operand
__device__ __forceinline__ float qt_rest(float x) { return x - __half2float(__float2half_rn(x)); }
__device__ __forceinline__ uint32_t qt_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
// log2 of a positive scale, exact for powers of two
__device__ __forceinline__ float qt_log2(float s) {
  const uint32_t bits = __float_as_uint(s);
  const float part = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
  const float e = (float)((int)((bits >> 23) & 0xff) - 127);
  return (bits & 0x7fffffu) ? e + __log2f(part) : e;
}
template <int kBytes>
__device__ __forceinline__ void qt_fetch(uint32_t to, const void* from, bool there) {
  const int n = there ? kBytes : 0;         // the rest is zeros
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(from), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;\n" ::"r"(to), "l"(from), "r"(n), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void qt_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void qt_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(kPending) : "memory");
}

template <int DP>
struct QtShape {
  static constexpr int kRow = DP;                         // bytes of a staged row
  static constexpr int kTile = 16 * kRow;
  static constexpr int kStage = 2 * kTile + 128;          // K, V, the tokens' scales
  static constexpr int kRing = QT_STAGES * kStage;
  static constexpr int kKey = DP >= 64 ? DP / 64 : 1;     // key pieces of a lane
  static constexpr int kKeyWords = DP >= 64 ? 4 : 2;      // of such a piece
  static constexpr int kWords = DP / 32;                  // value words of a lane and token
  static constexpr int kSum = DP + 4;                     // row of the joined sums (floats)
  // Pieces of 16 bytes change places within their 128-byte line, by the row, so that
  // the eight lanes of a read's phase meet all banks: for keys rows 0 and 1 (widths
  // below 128 lie side by side already), for values rows 0, 2, 4 and 6.
  static __device__ __forceinline__ int key_at(int row, int byte) {
    const int flip = DP >= 128 ? (row & 1) << 6 : 0;
    return row * kRow + (byte ^ flip);
  }
  static __device__ __forceinline__ int value_at(int row, int byte) {
    const int flip = DP >= 64 ? (row & 6) << 4 : (row & 4) << 3;
    return (row * kRow + byte) ^ flip;
  }
};

// A warp's work on one sequence and kTiles * 8 query heads, kSub tiles of 16 tokens a step.
template <typename T, int DP, int kTiles, int kSub>
struct QtState {
  using S = QtShape<DP>;
  static constexpr bool kSplit = std::is_same<T, float>::value;   // operands in two f16 parts
  static constexpr int kParts = kSplit ? 2 : 1, kHeads = 8 * kTiles;
  static constexpr int kSteps = S::kKey * S::kKeyWords;   // products of the scores
  uint32_t qf[kTiles][kSteps][2][kParts];
  float unit[kTiles][2];                    // of heads 2t, 2t + 1: log2(e) scale / 2^k
  float acc[kTiles][2 * S::kWords][4];      // columns (d, d + 1) x heads (2t, 2t + 1)
  float m[kTiles][2], l[kTiles][2];         // maxima and sums of the scores' weights
  float w_top[kTiles][2];                   // maxima of the scores with the value scale

  // Elements of a query row in the order of its pieces, as they come.
  struct Query {
    static constexpr int kEach = 16 / sizeof(T), kLoads = 4 * S::kKeyWords / kEach;
    uint4 words[kTiles][S::kKey][kLoads];
  };
  __device__ __forceinline__ static void fetch(const QuantArgs& a, int b, int head0, int n_heads,
                                               Query& query) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      const bool on = 8 * n + g < n_heads;
      const T* q = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb +
                   (int64_t)(head0 + (on ? 8 * n + g : 0)) * a.q_sh;
#pragma unroll
      for (int i = 0; i < S::kKey; ++i)
#pragma unroll
        for (int e = 0; e < Query::kLoads; ++e) {
          const int d = (t + 4 * i) * 4 * S::kKeyWords + e * Query::kEach;
          uint4& to = query.words[n][i][e];
          to = make_uint4(0, 0, 0, 0);
          if (!on || d >= a.D) continue;
          if (a.q_whole) {
            to = *reinterpret_cast<const uint4*>(q + d);
          } else {
            T* x = reinterpret_cast<T*>(&to);
#pragma unroll
            for (int c = 0; c < Query::kEach; ++c) x[c] = q[d + c];
          }
        }
    }
  }

  // Queries of head g, scaled by a power of two to at most 2^14: f16 then holds a
  // bf16 element down to 2^-25 of the head's largest exactly, and two parts hold
  // fp32 to 2^-22.
  __device__ __forceinline__ void begin(const QuantArgs& a, const Query& query) {
    const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      float x[S::kKey][4 * S::kKeyWords], top = 0.f;
#pragma unroll
      for (int i = 0; i < S::kKey; ++i) {
#pragma unroll
        for (int e = 0; e < 4 * S::kKeyWords; ++e) {
          const uint4& from = query.words[n][i][e / Query::kEach];
          const int c = e % Query::kEach;
          const uint32_t* w = reinterpret_cast<const uint32_t*>(&from);
          if constexpr (sizeof(T) == 4)
            x[i][e] = __uint_as_float(w[c]);
          else
            x[i][e] = __uint_as_float(c & 1 ? w[c / 2] & 0xffff0000u : w[c / 2] << 16);
          const float y = fabsf(x[i][e]);
          if (y <= 3.402823466e38f) top = fmaxf(top, y);
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      int k = top > 0.f ? 13 + 127 - (int)(__float_as_uint(top) >> 23) : 0;
      k = max(min(k, 120), -120);
      const float lift = __uint_as_float((uint32_t)(k + 127) << 23);
  #pragma unroll
      for (int i = 0; i < S::kKey; ++i)
  #pragma unroll
        for (int e = 0; e < 4 * S::kKeyWords; e += 4)
  #pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float u = x[i][e + 2 * c] * lift, v = x[i][e + 2 * c + 1] * lift;
            uint32_t (&to)[kParts] = qf[n][i * S::kKeyWords + e / 4][c];
            to[0] = qt_pack(u, v);
            if constexpr (kSplit) to[1] = qt_pack(qt_rest(u), qt_rest(v));
          }
      const float back = a.scale_log2 * __uint_as_float((uint32_t)(127 - k) << 23);
  #pragma unroll
      for (int r = 0; r < 2; ++r) unit[n][r] = __shfl_sync(0xffffffffu, back, (2 * t + r) * 4);
    }

#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
      for (int j = 0; j < 2 * S::kWords; ++j)
        acc[n][j][0] = acc[n][j][1] = acc[n][j][2] = acc[n][j][3] = 0.f;
#pragma unroll
      for (int r = 0; r < 2; ++r) m[n][r] = w_top[n][r] = QT_UNSET, l[n][r] = 0.f;
    }
  }

  // The staged tiles at `keys` and `values`; key scale and log2 of the value scale of
  // tokens g and g + 8 of each.
  __device__ __forceinline__ void step(const uint8_t* keys, const uint8_t* values,
                                       const uint32_t (&key)[kSub][2],
                                       const float (&value)[kSub][2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float s[kSub][kTiles][4];               // tokens (g, g + 8) x heads (2t, 2t + 1)
    float x[kSub][kTiles][4], z[kSub][kTiles][4];   // their exponents, without and with the
    bool grown = false;                             // value scale, above the references
    const auto exponents = [&](int u, bool above) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const bool there = key[u][r] != QT_ABSENT;
        const float scale = there ? __uint_as_float(key[u][r]) : 0.f, base = there ? 0.f : -INFINITY;
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float f = unit[n][c] * scale;
            x[u][n][2 * r + c] = fmaf(s[u][n][2 * r + c], f, above ? base - m[n][c] : base);
            z[u][n][2 * r + c] =
                fmaf(s[u][n][2 * r + c], f,
                     above ? (base + value[u][r]) - (w_top[n][c] - QT_LIFT) : base + value[u][r]);
          }
      }
    };
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
#pragma unroll
      for (int n = 0; n < kTiles; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.f;
#pragma unroll
      for (int i = 0; i < S::kKey; ++i) {
        uint32_t k[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint8_t* at = keys + u * S::kTile;
          if constexpr (DP >= 64) {
            const uint4 x = *reinterpret_cast<const uint4*>(at + S::key_at(g + 8 * r, 16 * (t + 4 * i)));
            k[r][0] = x.x, k[r][1] = x.y, k[r][2] = x.z, k[r][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(at + S::key_at(g + 8 * r, 8 * t));
            k[r][0] = x.x, k[r][1] = x.y;
          }
        }
#pragma unroll
        for (int e = 0; e < S::kKeyWords; ++e) {
          uint32_t f[4];
          qt_widen(k[0][e], f[0], f[2]);
          qt_widen(k[1][e], f[1], f[3]);
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
              const auto& q = qf[n][i * S::kKeyWords + e];
              qt_mma(s[u][n], f, q[0][p], q[1][p]);
            }
        }
      }
      exponents(u, true);
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          grown |= x[u][n][c] > QT_SLACK || z[u][n][c] > QT_LIFT + QT_SLACK;
    }
    if (__any_sync(0xffffffffu, grown)) {   // new references: the largest so far
#pragma unroll
      for (int u = 0; u < kSub; ++u) exponents(u, false);
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = m[n][c], high = w_top[n][c];
#pragma unroll
          for (int u = 0; u < kSub; ++u) {
            top = fmaxf(top, fmaxf(x[u][n][c], x[u][n][c + 2]));
            high = fmaxf(high, fmaxf(z[u][n][c], z[u][n][c + 2]));
          }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
          }
          l[n][c] *= qt_exp2(m[n][c] - top);
          const float keep = qt_exp2(w_top[n][c] - high);
#pragma unroll
          for (int j = 0; j < 2 * S::kWords; ++j) {
            acc[n][j][c] *= keep;
            acc[n][j][c + 2] *= keep;
          }
          m[n][c] = top;
          w_top[n][c] = high;
        }
#pragma unroll
      for (int u = 0; u < kSub; ++u) exponents(u, true);
    }
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      uint32_t p[kTiles][2][kParts];        // weights of tokens 2t, 2t + 1 (+ 8) of head g
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        float w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          l[n][c & 1] += qt_exp2(x[u][n][c]);
          w[c] = qt_exp2(z[u][n][c]);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          p[n][r][0] = qt_transpose(qt_pack(w[2 * r], w[2 * r + 1]));
          if constexpr (kSplit)
            p[n][r][1] = qt_transpose(qt_pack(qt_rest(w[2 * r]), qt_rest(w[2 * r + 1])));
        }
      }
      // values of tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
      for (int i = 0; i < (DP + 127) / 128; ++i) {
        constexpr int kRead = S::kWords < 4 ? S::kWords : 4;   // words of a read
        uint32_t v[4][kRead];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint8_t* x = values + u * S::kTile +
                             S::value_at(2 * t + (n & 1) + 8 * (n >> 1), 128 * i + 4 * kRead * g);
          if constexpr (kRead == 4) {
            const uint4 y = *reinterpret_cast<const uint4*>(x);
            v[n][0] = y.x, v[n][1] = y.y, v[n][2] = y.z, v[n][3] = y.w;
          } else if constexpr (kRead == 2) {
            const uint2 y = *reinterpret_cast<const uint2*>(x);
            v[n][0] = y.x, v[n][1] = y.y;
          } else {
            v[n][0] = *reinterpret_cast<const uint32_t*>(x);
          }
        }
#pragma unroll
        for (int e = 0; e < kRead; ++e)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const unsigned pick = c ? 0x7362u : 0x5140u;
            uint32_t f[4];
            qt_widen(__byte_perm(v[0][e], v[1][e], pick), f[0], f[1]);
            qt_widen(__byte_perm(v[2][e], v[3][e], pick), f[2], f[3]);
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
              for (int k = 0; k < kParts; ++k)
                qt_mma(acc[n][2 * (4 * i + e) + c], f, p[n][0][k], p[n][1][k]);
          }
      }
    }
  }

  // Every lane's share of the weights' sums, of all tokens.
  __device__ __forceinline__ void sum_weights() {
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], o);
  }
};

// Four warps on one slice of a sequence and K/V head, every fourth tile each, joined in
// shared memory: one launch for few tokens (5 sequences of 129 tokens 4.7 us, of which
// most is the chain length, look-up, copy, product).  kRuns: pages are multiples of 8.
template <typename T, int DP, int kTiles, int kPiece, bool kRuns>
__global__ void __launch_bounds__(32 * QT_WARPS) quant_mma_kernel(QuantArgs a) {
  using S = QtShape<DP>;
  constexpr int kHeads = 8 * kTiles;
  extern __shared__ __align__(128) uint8_t qt_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int chunks = (a.group + kHeads - 1) / kHeads;
  const int b = blockIdx.x / (a.kv_heads * chunks), h = blockIdx.x / chunks % a.kv_heads;
  const int head0 = h * a.group + blockIdx.x % chunks * kHeads;
  const int n_heads = min(kHeads, (h + 1) * a.group - head0);
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");

  const int past = quant_length(a, b), tiles = (past + 15) / 16;
  const int lo = (int)((int64_t)tiles * blockIdx.y / gridDim.y);
  const int hi = (int)((int64_t)tiles * (blockIdx.y + 1) / gridDim.y);
  const int mine = max(0, (hi - lo - warp + QT_WARPS - 1) / QT_WARPS);   // this warp's tiles
  typename QtState<T, DP, kTiles, 1>::Query query;
  QtState<T, DP, kTiles, 1>::fetch(a, b, head0, n_heads, query);
  uint8_t* ring = qt_smem + warp * S::kRing;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const int32_t* table = a.bt + (int64_t)b * a.bt_s;
  const uint8_t* const kh = a.kc + h * a.c_sh;
  const uint8_t* const vh = a.vc + h * a.c_sh;
  constexpr int kLanes = DP / kPiece, kRows = 32 / kLanes;   // lanes of a row, rows of a round
  const int lane_row = lane / kLanes, byte = lane % kLanes * kPiece;
  const bool inside = byte < a.D;
  const auto tile_of = [&](int j) { return lo + warp + j * QT_WARPS; };
  const auto column = [&](int token) {
    return a.magic ? (int)(__umulhi((uint32_t)token, a.magic) >> a.shift) : token;
  };

  // kRuns (pages of whole runs of 8 tokens): lane i looks up the two runs of sixteen
  // tiles ahead at once - place, key scale and log2 of the value scale - and they are
  // handed round by shuffles; `next` is requested in steps while `now` is in use.
  // Else lanes i and i + 16 look up token i of the next tile to be requested.
  struct Runs {
    int64_t at;
    uint32_t key;
    float value;
  };
  int page = -1;
  const auto look = [&](int j) {             // the page of this lane's run, or token
    const int token = kRuns ? tile_of(j + (lane >> 1)) * 16 + (lane & 1) * 8
                            : tile_of(j) * 16 + (lane & 15);
    const bool ask = kRuns ? j + (lane >> 1) < mine : j < mine;
    page = ask && token < past ? __ldg(table + column(token)) : -1;
    return ask && token < past ? token : -1;
  };
  const auto place = [&](int token) {        // of the page looked up; -1: there is none
    const bool there = page >= 0 && page < a.pages;
    if (token >= 0 && !there) set_status(a.status, GRS_ERR_BAD_PAGE);
    return there ? (int64_t)page * a.c_sp + (int64_t)(token - column(token) * a.page) * a.c_st
                 : -1;
  };
  const auto scales_of = [&](Runs& r) {
    const int64_t at = (int64_t)page * a.s_sp + h;
    r.key = r.at >= 0 ? __float_as_uint(__ldg(a.ks + at)) : QT_ABSENT;
    r.value = r.at >= 0 ? __ldg(a.vs + at) : 0.f;
  };
  Runs now = {}, next = {};
  int token = look(0);
  if constexpr (kRuns) {
    now.at = place(token);
    scales_of(now);
    token = look(16);
    next.at = place(token);
    scales_of(next);
    now.value = qt_log2(now.value);
    next.value = qt_log2(next.value);
  }
  int batch = 0;                             // first tile of `now`
  const auto request = [&](int j, int stage) {
    if (j >= mine) {
      qt_commit();
      return;
    }
    const int left = past - tile_of(j) * 16; // tokens of this tile
    const uint32_t base = ring_at + stage * S::kStage;
    int64_t at;
    if constexpr (kRuns) {
      at = j - batch < 16 ? now.at : next.at;
    } else {
      at = place(token);
      // scales: the keys' by the first 16 lanes, the values' by the others
      const uint32_t scale = base + 2 * S::kTile + 4 * lane;
      if (at >= 0)
        qt_fetch<4>(scale, (lane < 16 ? a.ks : a.vs) + page * a.s_sp + h, true);
      else
        asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(scale), "r"(lane < 16 ? QT_ABSENT : 0u)
                     : "memory");
    }
#pragma unroll
    for (int i = 0; i < 16 / kRows; ++i) {
      const int row = i * kRows + lane_row;
      int64_t from;
      bool fetch = inside;
      if constexpr (kRuns) {
        from = __shfl_sync(0xffffffffu, at, ((j & 15) << 1) + (row >> 3));
        fetch = fetch && from >= 0 && row < left;
        from += (row & 7) * a.c_st;
      } else {
        from = __shfl_sync(0xffffffffu, at, row);
        fetch = fetch && from >= 0;
      }
      from = fetch ? from + byte : 0;
      qt_fetch<kPiece>(base + S::key_at(row, byte), kh + from, fetch);
      qt_fetch<kPiece>(base + S::kTile + S::value_at(row, byte), vh + from, fetch);
    }
    qt_commit();
    if constexpr (!kRuns) token = look(j + 1);
  };
#pragma unroll
  for (int i = 0; i < QT_STAGES - 1; ++i) request(i, i);

  QtState<T, DP, kTiles, 1> state;
  state.begin(a, query);
  int stage = 0;
  for (int j = 0; j < mine; ++j) {
    if constexpr (kRuns) {
      // the last tiles' requests are ahead in `next`; the one after it is looked up in
      // three steps, so that no load is waited for
      const int at = j & 15;
      if (at == 0 && j > 0) {
        now = next;
        batch = j;
        token = look(j + 16);
      } else if (at == 4 && j > 16) {
        next.at = place(token);
        scales_of(next);
      } else if (at == 8 && j > 16) {
        next.value = qt_log2(next.value);
      }
    }
    qt_wait<QT_STAGES - 2>();
    __syncwarp();
    request(j + QT_STAGES - 1, stage == 0 ? QT_STAGES - 1 : stage - 1);
    const uint8_t* at = ring + stage * S::kStage;
    stage = stage + 1 == QT_STAGES ? 0 : stage + 1;

    const uint32_t* scales = reinterpret_cast<const uint32_t*>(at + 2 * S::kTile);
    const int left = past - tile_of(j) * 16;
    uint32_t key[1][2];
    float value[1][2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (kRuns) {
        key[0][r] = __shfl_sync(0xffffffffu, now.key, ((j & 15) << 1) + r);
        value[0][r] = __shfl_sync(0xffffffffu, now.value, ((j & 15) << 1) + r);
        if (g + 8 * r >= left) key[0][r] = QT_ABSENT;
      } else {
        key[0][r] = scales[g + 8 * r];
        value[0][r] = qt_log2(__uint_as_float(scales[16 + g + 8 * r]));
      }
    }
    state.step(at, at + S::kTile, key, value);
  }

  // the warps' sums meet in shared memory
  qt_wait<0>();
  __syncthreads();
  float* sums = reinterpret_cast<float*>(qt_smem);        // [warps][kHeads][kSum]
  float* tops = sums + QT_WARPS * kHeads * S::kSum;       // [warps][kHeads][3]
  state.sum_weights();
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int head = 8 * n + 2 * t + r;
      float* row = sums + (warp * kHeads + head) * S::kSum;
      constexpr int kRead = S::kWords < 4 ? S::kWords : 4;
#pragma unroll
      for (int j = 0; j < S::kWords; ++j)
        *reinterpret_cast<float4*>(row + 128 * (j / 4) + 4 * kRead * g + 4 * (j % 4)) = make_float4(
            state.acc[n][2 * j][r], state.acc[n][2 * j][r + 2], state.acc[n][2 * j + 1][r],
            state.acc[n][2 * j + 1][r + 2]);
      if (g == 0) {
        float* top = tops + (warp * kHeads + head) * 3;
        top[0] = state.m[n][r];
        top[1] = state.l[n][r];
        top[2] = state.w_top[n][r];
      }
    }
  __syncthreads();
  const int64_t stride = (int64_t)a.batch * a.heads;
  for (int head = warp; head < n_heads; head += QT_WARPS) {
    float top = QT_UNSET, high = QT_UNSET;
#pragma unroll
    for (int i = 0; i < QT_WARPS; ++i) {
      top = fmaxf(top, tops[(i * kHeads + head) * 3]);
      high = fmaxf(high, tops[(i * kHeads + head) * 3 + 2]);
    }
    const float base = top == QT_UNSET ? 0.f : top, w_base = high == QT_UNSET ? 0.f : high;
    float norm = 0.f, w[QT_WARPS];
#pragma unroll
    for (int i = 0; i < QT_WARPS; ++i) {
      const float* x = tops + (i * kHeads + head) * 3;
      norm = fmaf(exp2f(x[0] - base), x[1], norm);
      w[i] = exp2f(x[2] - w_base);
    }
    // the references' difference in two halves: either alone may leave the range
    const float half = exp2f(0.5f * (w_base - base - QT_LIFT));
    const float inv = norm == 0.f ? 0.f : half / norm;
    const int64_t row = (int64_t)b * a.heads + head0 + head;
    for (int d = 4 * lane; d < a.D; d += 128) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < QT_WARPS; ++i) {
        const float4 y =
            *reinterpret_cast<const float4*>(sums + (i * kHeads + head) * S::kSum + d);
        x.x = fmaf(w[i], y.x, x.x);
        x.y = fmaf(w[i], y.y, x.y);
        x.z = fmaf(w[i], y.z, x.z);
        x.w = fmaf(w[i], y.w, x.w);
      }
      const float o[4] = {x.x * inv * half, x.y * inv * half, x.z * inv * half, x.w * inv * half};
      if (a.slices > 1) {
        *reinterpret_cast<float4*>(a.part + (blockIdx.y * stride + row) * a.D + d) =
            make_float4(o[0], o[1], o[2], o[3]);
      } else {
        T* to = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)(head0 + head) * a.o_sh + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = from_float<T>(o[i]);
      }
    }
    if (a.slices > 1 && lane == 0)
      a.part_lse[blockIdx.y * stride + row] = norm == 0.f ? -INFINITY : base + log2f(norm);
  }
}

// ---- long contexts: a stream of tiles per warp -----------------------------------
// The tiles of all sequences in a row are cut into as many equal ranges as the SMs hold
// warps for each K/V head, whatever the sequences' lengths; a warp goes through its
// range of one head, from one sequence into the next without draining its ring, and
// the warps of the other heads of those tokens run beside it, so that whole pages are
// read at once.  A sequence that one range holds is written at once; parts of one go to
// the workspace, at most two of a range, and are joined by quant_join_kernel.  Two, three
// or five ranges a warp balance no better than their starts cost (73, 79, 91 us against 63).
// bf16, 32/8 heads of 128: 64 sequences of 300 to 4099 tokens 60 us (310 MB, 5.2 TB/s; 55 %
// of the issue slots), 512 of 2048 to 4096 484 us = 6.6 TB/s, a plain copy's rate (568, 5.6
// TB/s, after 40 ms of load and more: the clocks sink under the power limit), 2 of up to
// 131000 86 to 94 us.  Narrow heads and fp32 are bound by instructions: 200 sequences of up
// to 1001 tokens of 8 heads of 32 take 27 us in bf16 and 29 to 30 in fp32, which HBM would
// read in 6 to 8 (249 and 275 a tile; fp32 spills 108 bytes at the 96 registers of five CTAs).
constexpr int QS_SHORT = 1024;              // tokens of a table row that one warp takes
constexpr int QS_MOST = 1024;               // sequences: their first tiles are in shared memory
// (1024 of 300 to 2000 tokens 385 us by ranges, 1025 in slices of four warps 397)

template <typename T, int DP, int kTiles>
struct QsShape {
  // CTAs that share an SM (by registers), tokens of a step, steps that a warp has in
  // flight and in use: fewer warps with more steps in flight read faster (64 sequences of
  // up to 4099 tokens: four CTAs of three 16-token steps 63 us, three of four 61.5)
  static constexpr bool kSplit = std::is_same<T, float>::value;
  static constexpr int kCtas = DP > 128 ? 2 : DP > 64 ? (kTiles == 1 ? 3 : 2)
                             : kTiles == 1 ? (DP > 32 ? 4 : 5) : kSplit ? 2 : 3;
  static constexpr int kSub = DP > 64 || kTiles == 2 ? 1 : 2, kSpan = 16 * kSub;
  static constexpr int kStages = DP > 128 || (DP == 64 && kSub == 2) ? 3 : 4;
  static constexpr int kStage = 2 * kSub * QtShape<DP>::kTile;
  static constexpr int kBits = kSub == 1 ? 4 : 5;         // log2 of kSpan
};

// First steps of the sequences, shifted left by kBits, with the tokens of the last step
// (0: all) below; shared memory, `starts[batch]` is all steps.  Two barriers.
template <int kBits>
__device__ __forceinline__ void quant_starts(const QuantArgs& a, int* starts, int* sums) {
  constexpr int kThreads = 32 * QT_WARPS, kEach = QS_MOST / kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (a.batch + kThreads - 1) / kThreads, room = a.columns * a.page;
  int past[kEach], total = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int b = threadIdx.x * each + i;
    past[i] = 0;
    if (i < each && b < a.batch) {
      const int length = __ldg(a.lengths + b);
      past[i] = min(max(length, 0), room);
      if (blockIdx.x == 0 && past[i] != length) set_status(a.status, GRS_ERR_LENGTH);
      if (a.pages == 0 && past[i] > 0) {
        if (blockIdx.x == 0) set_status(a.status, GRS_ERR_BAD_PAGE);
        past[i] = 0;
      }
    }
    total += (past[i] + (1 << kBits) - 1) >> kBits;
  }
  int before = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  if (lane == 31) sums[warp] = before;
  __syncthreads();
  before -= total;
  for (int i = 0; i < warp; ++i) before += sums[i];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int b = threadIdx.x * each + i;
    if (i < each && b <= a.batch) starts[b] = before << kBits | (past[i] & ((1 << kBits) - 1));
    before += (past[i] + (1 << kBits) - 1) >> kBits;
  }
  if (threadIdx.x == kThreads - 1 && a.batch == kThreads * each) starts[a.batch] = before << kBits;
  __syncthreads();
}

// How all steps are cut: ranges of four steps at least, the first `rest` of them one
// longer than the others.
struct QsCut {
  int ranges, each, rest;
  __device__ __forceinline__ QsCut(int most, int total) {
    ranges = max(1, min(most, total / 4));
    each = total / ranges;
    rest = total - each * ranges;
  }
  __device__ __forceinline__ int first(int range) const { return each * range + min(range, rest); }
  __device__ __forceinline__ int holds(int tile) const {   // the range that does
    const int longer = rest * (each + 1);
    return tile < longer ? tile / (each + 1) : rest + (tile - longer) / each;
  }
};

template <typename T>
__device__ __forceinline__ void quant_store(T* to, const float (&x)[4], bool whole) {
  if (!whole) {
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = from_float<T>(x[i]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo),
                                               *reinterpret_cast<const uint32_t*>(&hi));
  }
}

// kWhole: every warp has one sequence (short ones; no table of first steps, no parts).
template <typename T, int DP, int kTiles, int kPiece, bool kWhole>
__global__ void __launch_bounds__(32 * QT_WARPS, (QsShape<T, DP, kTiles>::kCtas))
    quant_stream_kernel(QuantArgs a) {
  using S = QtShape<DP>;
  using Q = QsShape<T, DP, kTiles>;
  using State = QtState<T, DP, kTiles, Q::kSub>;
  constexpr int kHeads = 8 * kTiles, kStages = Q::kStages, kSub = Q::kSub, kBits = Q::kBits;
  constexpr int kAhead = 16 / kSub;          // steps that the lanes look up at once
  extern __shared__ __align__(128) uint8_t qt_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (!kWhole) asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  uint8_t* ring = qt_smem + warp * kStages * Q::kStage;
  const int* starts = reinterpret_cast<int*>(qt_smem + QT_WARPS * kStages * Q::kStage);
  const int chunks = (a.group + kHeads - 1) / kHeads, units = a.kv_heads * chunks;
  const int job = blockIdx.x * QT_WARPS + warp;
  const int range = job / units, part = job - range * units, h = part / chunks;
  const int head0 = h * a.group + part % chunks * kHeads;
  const int n_heads = min(kHeads, (h + 1) * a.group - head0);
  int lo, hi, seq = 0, whole_fill = 0;
  if constexpr (kWhole) {
    if (range >= a.batch) return;
    const int past = quant_length(a, range, true);
    seq = range;
    lo = 0;
    hi = (past + Q::kSpan - 1) >> kBits;
    whole_fill = past & (Q::kSpan - 1);
    if (hi == 0) {                           // no keys
      for (int i = lane; i < n_heads * a.D; i += 32)
        static_cast<T*>(a.out)[seq * a.o_sb + (head0 + i / a.D) * a.o_sh + i % a.D] =
            from_float<T>(0.f);
      return;
    }
  } else {
    quant_starts<kBits>(a, const_cast<int*>(starts), reinterpret_cast<int*>(qt_smem));
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i <= a.batch; i += 32 * QT_WARPS) a.starts[i] = starts[i] >> kBits;
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {     // rows without keys
      if (starts[b] >> kBits != starts[b + 1] >> kBits) continue;
      for (int h = warp; h < a.heads; h += QT_WARPS)            // (a row may pass 2^31 elements)
        for (int d = lane; d < a.D; d += 32)
          static_cast<T*>(a.out)[b * a.o_sb + h * a.o_sh + d] = from_float<T>(0.f);
    }
    const QsCut cut(a.ranges, starts[a.batch] >> kBits);
    if (range >= cut.ranges) return;
    lo = cut.first(range);
    hi = cut.first(range + 1);
    if (lo >= hi) return;
    for (int left = a.batch; left > 1;) {    // the last sequence that starts at or before lo
      const int half = left / 2;
      if (starts[seq + half] >> kBits <= lo) {
        seq += half;
        left -= half;
      } else {
        left = half;
      }
    }
  }
  const auto first_of = [&](int b) { return kWhole ? 0 : starts[b] >> kBits; };
  const auto last_of = [&](int b) { return kWhole ? hi : starts[b + 1] >> kBits; };
  int current = seq;                         // of the warp; seq: of this lane's look-ups
  typename State::Query query;
  State::fetch(a, current, head0, n_heads, query);

  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const uint8_t* const kh = a.kc + h * a.c_sh;
  const uint8_t* const vh = a.vc + h * a.c_sh;
  constexpr int kLanes = DP / kPiece, kRows = 32 / kLanes;   // lanes of a row, rows of a round
  const int lane_row = lane / kLanes, byte = lane % kLanes * kPiece;
  const bool inside = byte < a.D;
  const int64_t lane_at = (lane_row & 7) * a.c_st + byte;
  const int mine = hi - lo;

  // Lane i looks up one run of 8 tokens, all of them kAhead steps' at once - place, tokens
  // of the step, key scale and log2 of the value scale - and they are handed round by
  // shuffles; `next` is looked up in stages while `now` is in use.
  struct Runs {
    int64_t at;
    int left;
    uint32_t key;
    float value;
  };
  Runs now, next;
  int page = -1, token = -1;
  const auto look = [&](int j) {
    const int f = lo + j + lane / (2 * kSub);
    page = token = -1;
    next.left = 0;
    if (f >= hi) return;
    if constexpr (!kWhole)
      while (last_of(seq) <= f) ++seq;
    const int fill = kWhole ? whole_fill : starts[seq] & (Q::kSpan - 1);
    const int row = lane % (2 * kSub) * 8;
    next.left = f + 1 == last_of(seq) && fill ? fill : Q::kSpan;
    if (row >= next.left) return;
    token = (f - first_of(seq)) * Q::kSpan + row;
    const int column = a.magic ? (int)(__umulhi((uint32_t)token, a.magic) >> a.shift) : token;
    page = __ldg(a.bt + (int64_t)seq * a.bt_s + column);
    token -= column * a.page;                // the run's first row in its page
  };
  const auto place = [&] {
    const bool there = page >= 0 && page < a.pages;
    if (token >= 0 && !there) set_status(a.status, GRS_ERR_BAD_PAGE);
    next.at = there ? (int64_t)page * a.c_sp + (int64_t)token * a.c_st : -1;
    const int64_t at = (int64_t)page * a.s_sp + h;
    next.key = there ? __float_as_uint(__ldg(a.ks + at)) : QT_ABSENT;
    next.value = there ? __ldg(a.vs + at) : 0.f;
  };
  {
    look(0);                                 // the second look-up's pages with the first's
    const int page0 = page, token0 = token, left0 = next.left;
    look(kAhead);
    const int page1 = page, token1 = token, left1 = next.left;
    page = page0;
    token = token0;
    place();
    now = next;
    now.left = left0;
    page = page1;
    token = token1;
    place();
    next.left = left1;
    now.value = qt_log2(now.value);
    next.value = qt_log2(next.value);
  }
  int batch = 0;                             // first step of `now`
  const auto request = [&](int j, int stage) {
    if (j >= mine) {
      qt_commit();
      return;
    }
    const bool near = j - batch < kAhead;
    const int64_t at = near ? now.at : next.at;
    const int run0 = j % kAhead * 2 * kSub;
    const int left = __shfl_sync(0xffffffffu, near ? now.left : next.left, run0);
    const uint32_t base = ring_at + stage * Q::kStage;
#pragma unroll
    for (int i = 0; i < Q::kSpan / kRows; ++i) {
      const int row = i * kRows + lane_row, tile = row / 16 * S::kTile;
      // a lane's row in its run is the same in every round, or in every other one
      const int64_t shift = kRows % 8 == 0 ? lane_at : kRows == 4 ? lane_at + i % 2 * 4 * a.c_st
                                                                  : (row & 7) * a.c_st + byte;
      const int64_t from = __shfl_sync(0xffffffffu, at, run0 + (row >> 3));
      const bool fetch = inside && from >= 0 && row < left;
      const int64_t place = fetch ? from + shift : 0;
      qt_fetch<kPiece>(base + tile + S::key_at(row % 16, byte), kh + place, fetch);
      qt_fetch<kPiece>(base + kSub * S::kTile + tile + S::value_at(row % 16, byte), vh + place,
                       fetch);
    }
    qt_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) request(i, i);

  State state;
  // The next sequence of this range, whose queries are fetched under the current one's steps.
  int following = current;
  const auto begin = [&] {
    state.begin(a, query);
    if constexpr (!kWhole) {
      if (last_of(current) >= hi) return;
      following = current + 1;
      while (last_of(following) <= last_of(current)) ++following;
      State::fetch(a, following, head0, n_heads, query);
    }
  };
  begin();
  // Writes the current sequence's rows, or its part in this range.
  const auto finish = [&] {
    state.sum_weights();
    const bool whole = kWhole || (first_of(current) >= lo && last_of(current) <= hi);
    const int64_t slot = 2 * (int64_t)range + (first_of(current) >= lo ? 1 : 0);
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int head = 8 * n + 2 * t + r;
        if (head >= n_heads) continue;
        const float norm = state.l[n][r], top = state.m[n][r], high = state.w_top[n][r];
        const float base = top == QT_UNSET ? 0.f : top, w_base = high == QT_UNSET ? 0.f : high;
        // the references' difference in two halves: either alone may leave the range
        const float half = qt_exp2(0.5f * (w_base - base - QT_LIFT));
        const float inv = norm == 0.f ? 0.f : __fdividef(half, norm);
        const int64_t row = slot * a.heads + head0 + head;
        T* to = static_cast<T*>(a.out) + current * a.o_sb + (head0 + head) * a.o_sh;
        constexpr int kRead = S::kWords < 4 ? S::kWords : 4;
#pragma unroll
        for (int j = 0; j < S::kWords; ++j) {
          const int d = 128 * (j / 4) + 4 * kRead * g + 4 * (j % 4);
          if (d >= a.D) continue;
          const float x[4] = {state.acc[n][2 * j][r] * inv * half,
                              state.acc[n][2 * j][r + 2] * inv * half,
                              state.acc[n][2 * j + 1][r] * inv * half,
                              state.acc[n][2 * j + 1][r + 2] * inv * half};
          if (whole)
            quant_store<T>(to + d, x, a.o_whole);
          else
            quant_store<float>(a.part + row * a.D + d, x, true);
        }
        if (!whole && g == 0) a.part_lse[row] = norm == 0.f ? -INFINITY : base + log2f(norm);
      }
  };
  int end = min(last_of(current), hi) - lo, stage = 0;
  for (int j = 0; j < mine; ++j) {
    const int at = j % kAhead;
    if (at == 0 && j > 0) {
      now = next;
      batch = j;
      look(j + kAhead);
    } else if (at == kAhead / 4 && j > kAhead) {
      place();
    } else if (at == kAhead / 2 && j > kAhead) {
      next.value = qt_log2(next.value);
    }
    qt_wait<kStages - 2>();
    __syncwarp();
    request(j + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
    if (!kWhole && j == end) {
      finish();
      current = following;
      end = min(last_of(current), hi) - lo;
      begin();
    }
    const int left = __shfl_sync(0xffffffffu, now.left, at * 2 * kSub);
    uint32_t key[kSub][2];
    float value[kSub][2];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        key[u][r] = __shfl_sync(0xffffffffu, now.key, at * 2 * kSub + 2 * u + r);
        value[u][r] = __shfl_sync(0xffffffffu, now.value, at * 2 * kSub + 2 * u + r);
        if (16 * u + g + 8 * r >= left) key[u][r] = QT_ABSENT;
      }
    const uint8_t* keys = ring + stage * Q::kStage;
    state.step(keys, keys + kSub * S::kTile, key, value);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  finish();
}

// A row's partial sums joined by their weights: `team` (1 or 4) of a CTA's four warps per
// (sequence, head).  The parts are still in L2; the launch overlaps the end of the kernel
// before it, and adds about 4 us to 64 sequences of 32 heads of 128.
template <typename T>
__global__ void __launch_bounds__(128) quant_join_kernel(QuantArgs a, int team) {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  __shared__ float4 xs[4][32];
  __shared__ float norms[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rows = (int64_t)a.batch * a.heads;
  const int64_t row = team == 4 ? blockIdx.x : (int64_t)blockIdx.x * 4 + warp;
  if (row >= rows) return;                  // whole CTAs, or warps that meet nobody
  const int b = (int)(row / a.heads), head = (int)(row % a.heads);
  int parts = a.slices, first = 0;
  if (a.ranges) {
    const int total = a.starts[a.batch], from = a.starts[b], to = a.starts[b + 1];
    if (from == to) return;
    const QsCut cut(a.ranges, total);
    first = cut.holds(from);
    parts = cut.holds(to - 1) - first + 1;
    if (parts == 1) return;                 // written already
  }
  const auto at = [&](int i) {              // row of part i
    if (!a.ranges) return i * rows + row;
    return (2 * (int64_t)(first + i) + (i == 0 ? 1 : 0)) * a.heads + head;
  };
  const int step = team, mine0 = team == 4 ? warp : 0;
  // a lane's first part, before anything waits for the others'
  const float early = mine0 + lane * step < parts ? a.part_lse[at(mine0 + lane * step)] : -INFINITY;
  float top = early;
  if (step > 1 || parts > 32)
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, a.part_lse[at(i)]);
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  for (int d0 = 0; d0 < a.D; d0 += 128) {
    const int d = d0 + 4 * lane;
    float norm = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = mine0; p0 < parts; p0 += 32 * step) {
      const int mine = p0 + lane * step;
      const float lse = p0 == mine0 ? early : mine < parts ? a.part_lse[at(mine)] : -INFINITY;
      const float w = exp2f(lse - base);
      norm += warp_sum(w);
      const int n = min(32, (parts - p0 + step - 1) / step);
      for (int i0 = 0; i0 < n; i0 += 8) {
        float4 y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i0 + i < n && d < a.D)
            y[i] = *reinterpret_cast<const float4*>(a.part + at(p0 + (i0 + i) * step) * a.D + d);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float wi = __shfl_sync(0xffffffffu, w, min(i0 + i, 31));
          x.x = fmaf(wi, y[i].x, x.x);
          x.y = fmaf(wi, y[i].y, x.y);
          x.z = fmaf(wi, y[i].z, x.z);
          x.w = fmaf(wi, y[i].w, x.w);
        }
      }
    }
    if (team == 4) {
      if (d0) __syncthreads();              // the last columns' sums are read
      xs[warp][lane] = x;
      if (lane == 0) norms[warp] = norm;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i == warp) continue;
        const float4 y = xs[i][lane];
        x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        norm += norms[i];
      }
    }
    const float inv = norm == 0.f ? 0.f : 1.f / norm;
    const float o[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    if (d < a.D && (team == 1 || warp == 0))
      quant_store<T>(static_cast<T*>(a.out) + b * a.o_sb + head * a.o_sh + d, o, a.o_whole);
  }
}

template <typename T>
static int quant_join(const QuantArgs& p, int parts, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.batch * p.heads;
  const int team = parts > 8 ? 4 : 1;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(team == 4 ? rows : (rows + 3) / 4));
  config.blockDim = dim3(128);
  config.stream = counted(stream);
  config.attrs = &attr;
  config.numAttrs = 1;
  if (cudaLaunchKernelEx(&config, quant_join_kernel<T>, p, team) != cudaSuccess)
    return GRS_ERR_CUDA;
  GRS_CUDA_CHECK_LAUNCH();
  return GRS_OK;
}

// Whether a CTA takes 16 query heads of a group (two column tiles); above width 128
// their accumulators and queries would not fit the registers.
static bool quant_wide(int group, int D) { return group > 8 && D <= 128; }

// Slices of each sequence: enough CTAs to fill the SMs several times, at least 256
// tokens each (by the table's width: the lengths are on the device).
static int quant_slices(int batch, int heads, int kv_heads, int D, int64_t room) {
  const int group = heads / kv_heads, chunk = quant_wide(group, D) ? 16 : 8;
  const int64_t tasks = (int64_t)batch * kv_heads * ((group + chunk - 1) / chunk);
  const int64_t want = (4 * 3 * 148 + tasks - 1) / tasks;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, 128, room / 256}));
}

// Ranges of the stream form, or 0: sequences that fit its table, and steps enough to give
// the warps of all SMs (by the type and width, at most 20 an SM) several each, if the
// tables are full.  Otherwise four warps share a sequence's head: 5 sequences of 129
// tokens take one launch there.
static int quant_ranges(int batch, int heads, int kv_heads, int D, int64_t room, int warps) {
  const int group = heads / kv_heads, chunk = quant_wide(group, D) ? 16 : 8;
  const int64_t units = (int64_t)kv_heads * ((group + chunk - 1) / chunk);
  const int64_t tiles = batch * ((room + 15) / 16);
  if (batch > QS_MOST || tiles >= 1 << 26 || tiles * units < 4 * (int64_t)warps) return 0;
  return (int)std::max<int64_t>(1, std::min<int64_t>(warps / units, (tiles + 3) / 4));
}
// Whether a warp takes a whole sequence's head: short ones, enough of them (bf16; tokens
// are up to the number given; 32/8 heads of 128: 1000 sequences of 256 / 512 / 1000 tokens
// 58 / 98 / 181 us against 83 / 119 / 191 by ranges, 500 of 500 57 against 66, 200 of 1000
// 60 against 52; 14/2 heads of 40: 800 of 700 33 against 38; 40/4 heads of 64: 300 of 500
// 25 against 36; 8/8 heads of 32: 200 of 1000 31 against 27).  The table's width stands for
// the lengths, which are on the device: wider tables lose that difference.
static bool quant_whole(int batch, int heads, int kv_heads, int D, int64_t room) {
  const int group = heads / kv_heads, chunk = quant_wide(group, D) ? 16 : 8;
  const int64_t units = (int64_t)kv_heads * ((group + chunk - 1) / chunk);
  return room <= QS_SHORT && batch * units >= std::max<int64_t>(4 * 148, 2 * room);
}
template <typename T, int DP, int kTiles>
constexpr int quant_warps() { return 148 * QsShape<T, DP, kTiles>::kCtas * QT_WARPS; }

static bool quant_aligned(const QuantArgs& p, int bytes) {
  const uint64_t bits = reinterpret_cast<uintptr_t>(p.kc) | reinterpret_cast<uintptr_t>(p.vc) |
                        (uint64_t)p.c_sp | (uint64_t)p.c_st | (uint64_t)p.c_sh | (uint64_t)p.D;
  return bits % bytes == 0;
}

template <typename T, int DP, int kTiles, int kPiece, bool kRuns>
static int quant_mma_run(const QuantArgs& p, cudaStream_t stream) {
  using S = QtShape<DP>;
  constexpr int kSums = QT_WARPS * 8 * kTiles * (S::kSum + 3) * 4;
  constexpr int smem = std::max(QT_WARPS * S::kRing, kSums);
  const int chunks = (p.group + 8 * kTiles - 1) / (8 * kTiles);
  const int64_t tasks = (int64_t)p.batch * p.kv_heads * chunks;
  const int64_t rows = (int64_t)p.batch * p.heads;
  if (tasks > INT_MAX || rows > INT_MAX) return GRS_ERR_SHAPE;
  if (smem > 48 * 1024 && !allow_shared<quant_mma_kernel<T, DP, kTiles, kPiece, kRuns>>(smem))
    return GRS_ERR_CUDA;
  quant_mma_kernel<T, DP, kTiles, kPiece, kRuns>
      <<<dim3((unsigned)tasks, p.slices), 32 * QT_WARPS, smem, counted(stream)>>>(p);
  GRS_CUDA_CHECK_LAUNCH();
  if (p.slices > 1) return quant_join<T>(p, p.slices, stream);
  return GRS_OK;
}

template <typename T, int DP, int kTiles, int kPiece, bool kWhole>
static int quant_stream_run(QuantArgs p, cudaStream_t stream) {
  using Q = QsShape<T, DP, kTiles>;
  const int64_t units = (int64_t)p.kv_heads * ((p.group + 8 * kTiles - 1) / (8 * kTiles));
  constexpr int kRings = QT_WARPS * Q::kStages * Q::kStage;
  constexpr int kMostBytes = kRings + (kWhole ? 0 : (QS_MOST + 1) * 4);
  p.slices = 1;
  p.part_lse = p.part + 2 * (int64_t)p.ranges * p.heads * p.D;
  p.starts = reinterpret_cast<int32_t*>(p.part_lse + 2 * (int64_t)p.ranges * p.heads);
  if (kMostBytes > 48 * 1024 &&
      !allow_shared<quant_stream_kernel<T, DP, kTiles, kPiece, kWhole>>(kMostBytes))
    return GRS_ERR_CUDA;
  const int64_t jobs = units * (kWhole ? p.batch : p.ranges);
  if (jobs > INT_MAX - QT_WARPS || (int64_t)p.batch * p.heads > INT_MAX) return GRS_ERR_SHAPE;
  quant_stream_kernel<T, DP, kTiles, kPiece, kWhole>
      <<<(unsigned)((jobs + QT_WARPS - 1) / QT_WARPS), 32 * QT_WARPS,
         kRings + (kWhole ? 0 : (p.batch + 1) * 4), counted(stream)>>>(p);
  GRS_CUDA_CHECK_LAUNCH();
  return kWhole ? (int)GRS_OK : quant_join<T>(p, p.ranges / p.batch, stream);
}

template <typename T, int kTiles, int kPiece, bool kRuns>
static int quant_mma_width(const QuantArgs& p, cudaStream_t stream) {
  const auto go = [&](auto width, auto tiles) -> int {
    constexpr int DP = decltype(width)::value, kT = decltype(tiles)::value;
    if constexpr (kRuns) {
      const int64_t room = (int64_t)p.columns * p.page;
      if (quant_whole(p.batch, p.heads, p.kv_heads, p.D, room))
        return quant_stream_run<T, DP, kT, kPiece, true>(p, stream);
      QuantArgs q = p;
      q.ranges = quant_ranges(p.batch, p.heads, p.kv_heads, p.D, room, quant_warps<T, DP, kT>());
      if (q.ranges) return quant_stream_run<T, DP, kT, kPiece, false>(q, stream);
    }
    return quant_mma_run<T, DP, kT, kPiece, kRuns>(p, stream);
  };
  const std::integral_constant<int, kTiles> tiles;
  if (p.D <= 32) return go(std::integral_constant<int, 32>{}, tiles);
  if (p.D <= 64) return go(std::integral_constant<int, 64>{}, tiles);
  if (kTiles == 2 || p.D <= 128) return go(std::integral_constant<int, 128>{}, tiles);
  return go(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
}

template <typename T>
static int quant_launch(const QuantArgs& p, cudaStream_t stream) {
  if (quant_aligned(p, 8)) {
    const auto go = [&](auto tiles) -> int {
      constexpr int kTiles = decltype(tiles)::value;
      if (p.page % 8 == 0)
        return quant_aligned(p, 16) ? quant_mma_width<T, kTiles, 16, true>(p, stream)
                                    : quant_mma_width<T, kTiles, 8, true>(p, stream);
      return quant_mma_width<T, kTiles, 8, false>(p, stream);
    };
    return quant_wide(p.group, p.D) ? go(std::integral_constant<int, 2>{})
                                    : go(std::integral_constant<int, 1>{});
  }
  const int64_t rows = (int64_t)p.batch * p.heads;
  if (rows > INT_MAX) return GRS_ERR_SHAPE;
  quant_rows_kernel<T><<<(unsigned)rows, 128, 0, counted(stream)>>>(p);
  GRS_CUDA_CHECK_LAUNCH();
  return GRS_OK;
}

}  // namespace grs

extern "C" int64_t grs_quantized_attention_workspace_bytes(int batch, int heads, int kv_heads,
                                                           int head_width, int64_t page_tokens) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 0;
  // any of the kernels may take the call, by the type and alignment of its tensors
  const int64_t slices = grs::quant_slices(batch, heads, kv_heads, head_width, page_tokens);
  int64_t words = slices > 1 ? slices * batch * heads * (head_width + 1) : 0;
  for (int warps = 148 * 2 * grs::QT_WARPS; warps <= 148 * 7 * grs::QT_WARPS; warps += 148 * grs::QT_WARPS) {
    const int64_t ranges =
        grs::quant_ranges(batch, heads, kv_heads, head_width, page_tokens, warps);
    if (ranges)
      words = std::max(words, 2 * ranges * heads * (head_width + 1) + batch + 1);
  }
  return words * 4;
}

extern "C" int grs_quantized_attention(
    int dtype, const void* query, int64_t q_sb, int64_t q_sh, const void* key_cache,
    const void* value_cache, int64_t c_sp, int64_t c_st, int64_t c_sh, const float* key_scale,
    const float* value_scale, int64_t s_sp, const int32_t* block_table, int64_t bt_stride,
    int max_blocks, const int32_t* lengths, int num_pages, int page_size, void* output,
    int64_t o_sb, int64_t o_sh, int batch, int heads, int kv_heads, int head_width, float scale,
    void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  using namespace grs;
  constexpr int kMost = 1 << 30;
  if ((dtype != GRS_DTYPE_F32 && dtype != GRS_DTYPE_BF16) || batch < 0 || batch >= kMost ||
      heads <= 0 || heads >= kMost || kv_heads <= 0 || heads % kv_heads || head_width <= 0 ||
      head_width > 256 || !std::isfinite(scale * QA_LOG2E) || max_blocks < 0 || num_pages < 0 ||
      page_size <= 0 || page_size >= kMost || (int64_t)max_blocks * page_size >= kMost)
    return GRS_ERR_SHAPE;
  if (batch == 0) return GRS_OK;
  if (!query || !output || !lengths || (max_blocks > 0 && !block_table) ||
      (num_pages > 0 && (!key_cache || !value_cache || !key_scale || !value_scale)))
    return GRS_ERR_SHAPE;
  const int64_t room = (int64_t)max_blocks * page_size;
  const int64_t need =
      grs_quantized_attention_workspace_bytes(batch, heads, kv_heads, head_width, room);
  if (need > 0 && (!workspace || workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return GRS_ERR_WORKSPACE;
  QuantArgs p = {};
  p.q = query; p.q_sb = q_sb; p.q_sh = q_sh;
  p.kc = static_cast<const uint8_t*>(key_cache); p.vc = static_cast<const uint8_t*>(value_cache);
  p.c_sp = c_sp; p.c_st = c_st; p.c_sh = c_sh;
  p.ks = key_scale; p.vs = value_scale; p.s_sp = s_sp;
  p.bt = block_table; p.bt_s = bt_stride; p.columns = max_blocks; p.lengths = lengths;
  p.pages = num_pages; p.page = page_size;
  if (page_size > 1) {                      // exact below 2^31 (round-up method)
    while ((1ll << (p.shift + 1)) < page_size) ++p.shift;
    p.magic = (uint32_t)(((1ull << (32 + p.shift)) + page_size - 1) / page_size);
  }
  const int item = dtype == GRS_DTYPE_F32 ? 4 : 2;
  p.q_whole = ((reinterpret_cast<uintptr_t>(query) | (uint64_t)(q_sb * item) |
                (uint64_t)(q_sh * item) | (uint64_t)(head_width * item)) & 15) == 0;
  p.o_whole = ((reinterpret_cast<uintptr_t>(output) | (uint64_t)(o_sb * item) |
                (uint64_t)(o_sh * item)) & (4 * item - 1)) == 0;
  p.slices = quant_slices(batch, heads, kv_heads, head_width, room);
  p.part = static_cast<float*>(workspace);
  p.part_lse = p.part + (int64_t)p.slices * batch * heads * head_width;
  p.out = output; p.o_sb = o_sb; p.o_sh = o_sh;
  p.batch = batch; p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads;
  p.D = head_width; p.scale_log2 = scale * QA_LOG2E; p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == GRS_DTYPE_F32 ? quant_launch<float>(p, s) : quant_launch<__nv_bfloat16>(p, s);
}
