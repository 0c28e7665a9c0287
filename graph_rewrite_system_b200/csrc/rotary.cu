// Rotary positions of packed queries and keys: grs_rotate_positions.
#include <algorithm>
#include <climits>
#include <cmath>

#include "rotary.cuh"

namespace grs {

struct RotateArgs {
  const void* q; int64_t q_st, q_sh; void* qo; int64_t qo_st, qo_sh; int heads;
  const void* k; int64_t k_st, k_sh; void* ko; int64_t ko_st, ko_sh; int kv_heads;
  const void* positions; int wide;          // int32 or int64 [tokens]
  const double* freq; int pairs; float magnitude;
  int tokens, width, rows;                  // tokens of a CTA
};

constexpr int ROT_THREADS = 256;
constexpr int ROT_AHEAD = 4;                // units of a thread in flight

// One CTA per `rows` tokens.  The (cos, sin) of its tokens' pairs are computed once
// into shared memory and serve every head; then each thread moves units (two
// pieces of 16 bytes that turn together) of one place in the head through the
// (token, head) rows, four at a time.
template <typename T, int kVec, bool kInter>
__global__ void __launch_bounds__(ROT_THREADS) rotate_kernel(RotateArgs a) {
  using Units = RotaryUnits<kVec, kInter>;
  using Piece = RotaryPiece<T, kVec>;
  extern __shared__ float2 rot_turns[];
  const int64_t first = (int64_t)blockIdx.x * a.rows;
  const int n = (int)min((int64_t)a.rows, a.tokens - first);
  for (int i = threadIdx.x; i < n * a.pairs; i += ROT_THREADS) {
    const int64_t at = first + i / a.pairs;
    const int64_t p = a.wide ? static_cast<const int64_t*>(a.positions)[at]
                             : static_cast<const int32_t*>(a.positions)[at];
    const float2 t = rotary_cos_sin(rotary_phase(p, rotary_step(a.freq[i % a.pairs])));
    rot_turns[i] = make_float2(t.x * a.magnitude, t.y * a.magnitude);
  }
  __syncthreads();

  const int units = Units::count(a.width, a.pairs), each = ROT_THREADS / units;
  const int all = a.heads + a.kv_heads;
  if (threadIdx.x >= each * units) return;
  const Units unit(threadIdx.x % units, a.pairs);
  int head = threadIdx.x / units % all, token = threadIdx.x / units / all;
  while (token < n) {
    Piece x[ROT_AHEAD], y[ROT_AHEAD];
    T* to[ROT_AHEAD];
    const float2* turns[ROT_AHEAD];
#pragma unroll
    for (int j = 0; j < ROT_AHEAD; ++j) {
      to[j] = nullptr;
      if (token >= n) continue;
      const bool key = head >= a.heads;
      const int64_t at = first + token, h = key ? head - a.heads : head;
      const T* from = key ? static_cast<const T*>(a.k) + at * a.k_st + h * a.k_sh
                          : static_cast<const T*>(a.q) + at * a.q_st + h * a.q_sh;
      to[j] = key ? static_cast<T*>(a.ko) + at * a.ko_st + h * a.ko_sh
                  : static_cast<T*>(a.qo) + at * a.qo_st + h * a.qo_sh;
      turns[j] = rot_turns + token * a.pairs + unit.pair;
      x[j] = *reinterpret_cast<const Piece*>(from + unit.a);
      if (unit.two()) y[j] = *reinterpret_cast<const Piece*>(from + unit.b);
      for (head += each; head >= all; head -= all) ++token;
    }
#pragma unroll
    for (int j = 0; j < ROT_AHEAD; ++j) {
      if (!to[j]) continue;
      if (unit.pair >= 0) {
        float u[kVec], v[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          u[i] = to_float(x[j].e[i]);
          v[i] = Units::kTwo ? to_float(y[j].e[i]) : 0.f;
        }
        rotary_turn<T, kVec, kInter>(turns[j], u, v);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          x[j].e[i] = from_float<T>(u[i]);
          y[j].e[i] = from_float<T>(v[i]);
        }
      }
      *reinterpret_cast<Piece*>(to[j] + unit.a) = x[j];
      if (unit.two()) *reinterpret_cast<Piece*>(to[j] + unit.b) = y[j];
    }
  }
}

template <typename T>
static int rotate_run(RotateArgs a, bool interleaved, cudaStream_t stream) {
  const int e = sizeof(T);
  int alignment = std::min(common_alignment(a.q, a.q_st * e, a.q_sh * e),
                           common_alignment(a.qo, a.qo_st * e, a.qo_sh * e));
  if (a.kv_heads)
    alignment = std::min({alignment, common_alignment(a.k, a.k_st * e, a.k_sh * e),
                          common_alignment(a.ko, a.ko_st * e, a.ko_sh * e)});
  // eight tokens share a table, fewer when that would leave SMs without a CTA
  a.rows = std::min(8, std::max(1, a.tokens / (4 * 148)));
  const int64_t ctas = ((int64_t)a.tokens + a.rows - 1) / a.rows;
  const int smem = a.rows * a.pairs * (int)sizeof(float2);
  return rotary_dispatch<T>(a.width, a.pairs, interleaved, alignment, [&](auto vec, auto inter) -> int {
    rotate_kernel<T, decltype(vec)::value, decltype(inter)::value>
        <<<(unsigned)ctas, ROT_THREADS, smem, counted(stream)>>>(a);
    GRS_CUDA_CHECK_LAUNCH();
    return GRS_OK;
  });
}

}  // namespace grs

extern "C" int grs_rotate_positions(
    int dtype, const void* query, int64_t q_st, int64_t q_sh, const void* key, int64_t k_st,
    int64_t k_sh, const void* positions, int positions_are_i64, const double* frequencies,
    int pairs, int interleaved, double magnitude, void* query_out, int64_t qo_st, int64_t qo_sh,
    void* key_out, int64_t ko_st, int64_t ko_sh, int tokens, int heads, int kv_heads,
    int head_width, void* stream) {
  using namespace grs;
  constexpr int kMost = 1 << 30;
  if (tokens < 0 || tokens >= kMost || heads <= 0 || heads >= kMost || kv_heads < 0 ||
      kv_heads >= kMost || head_width <= 0 || head_width > 256 || pairs <= 0 ||
      2 * pairs > head_width || !std::isfinite(magnitude))
    return GRS_ERR_SHAPE;
  if (tokens == 0) return GRS_OK;
  if (!query || !query_out || !positions || !frequencies || (kv_heads && (!key || !key_out)))
    return GRS_ERR_SHAPE;
  RotateArgs a = {};
  a.q = query; a.q_st = q_st; a.q_sh = q_sh; a.qo = query_out; a.qo_st = qo_st; a.qo_sh = qo_sh;
  a.k = key; a.k_st = k_st; a.k_sh = k_sh; a.ko = key_out; a.ko_st = ko_st; a.ko_sh = ko_sh;
  a.heads = heads; a.kv_heads = kv_heads;
  a.positions = positions; a.wide = positions_are_i64;
  a.freq = frequencies; a.pairs = pairs; a.magnitude = (float)magnitude;
  a.tokens = tokens; a.width = head_width;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == GRS_DTYPE_F32) return rotate_run<float>(a, interleaved != 0, s);
  if (dtype == GRS_DTYPE_BF16) return rotate_run<__nv_bfloat16>(a, interleaved != 0, s);
  return GRS_ERR_SHAPE;
}
