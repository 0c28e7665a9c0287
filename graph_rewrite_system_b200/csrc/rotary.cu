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

// One CTA per `rows` tokens.  The (cos, sin) of its tokens' pairs are computed once
// into shared memory; then every thread takes its own pairs' into registers and goes
// through the heads of its token (read from shared memory for every head: bank conflicts,
// 99 us against 58).  Bound by HBM: 16384 bf16 tokens of 32 + 8 heads of 128 (336 MB)
// take 58 us = 5.8 TB/s, 0.88 of a plain copy; one token 2.7 us.
template <typename T, int kVec, bool kInter>
__global__ void __launch_bounds__(ROT_THREADS, 3) rotate_kernel(RotateArgs a) {
  extern __shared__ __align__(16) float rot_turns[];
  const int64_t first = (int64_t)blockIdx.x * a.rows;
  const int n = (int)min((int64_t)a.rows, a.tokens - first);
  rotary_table<kVec, kInter, ROT_THREADS>(
      rot_turns, a.freq, a.pairs, a.magnitude, n, [&](int row) -> int64_t {
        return a.wide ? static_cast<const int64_t*>(a.positions)[first + row]
                      : static_cast<const int32_t*>(a.positions)[first + row];
      });
  __syncthreads();
  // one row of the grid for queries and one for keys, or one for both
  if (blockIdx.y == 0)
    rotary_rows<T, kVec, kInter, ROT_THREADS>(
        rot_turns, a.pairs, a.width, n, a.heads, static_cast<const T*>(a.q) + first * a.q_st,
        a.q_st, a.q_sh, static_cast<T*>(a.qo) + first * a.qo_st, a.qo_st, a.qo_sh);
  if (a.kv_heads && blockIdx.y == gridDim.y - 1)
    rotary_rows<T, kVec, kInter, ROT_THREADS>(
        rot_turns, a.pairs, a.width, n, a.kv_heads, static_cast<const T*>(a.k) + first * a.k_st,
        a.k_st, a.k_sh, static_cast<T*>(a.ko) + first * a.ko_st, a.ko_st, a.ko_sh);
}

template <typename T>
static int rotate_run(RotateArgs a, bool interleaved, cudaStream_t stream) {
  const int e = sizeof(T);
  int alignment = std::min(common_alignment(a.q, a.q_st * e, a.q_sh * e),
                           common_alignment(a.qo, a.qo_st * e, a.qo_sh * e));
  if (a.kv_heads)
    alignment = std::min({alignment, common_alignment(a.k, a.k_st * e, a.k_sh * e),
                          common_alignment(a.ko, a.ko_st * e, a.ko_sh * e)});
  return rotary_dispatch<T>(a.width, a.pairs, interleaved, alignment, [&](auto vec, auto inter) -> int {
    // tokens that share a CTA's table: eight, more of few heads (2048 units of work), fewer
    // when one wave of CTAs holds them all; up to 32 KB (12242 tokens of 6 heads of 96: 18
    // -> 8.7 us)
    const int units = RotaryUnits<decltype(vec)::value, decltype(inter)::value>::count(
        a.width, a.pairs);
    const int64_t work = (int64_t)(a.heads + a.kv_heads) * units;
    const int most = std::min((int)std::max<int64_t>(8, 2048 / work), std::min(64, 4096 / a.pairs));
    a.rows = std::min(most, (a.tokens + 3 * 148 - 1) / (3 * 148));
    const int64_t ctas = ((int64_t)a.tokens + a.rows - 1) / a.rows;
    const int smem = a.rows * a.pairs * 2 * (int)sizeof(float);
    rotate_kernel<T, decltype(vec)::value, decltype(inter)::value>
        <<<dim3((unsigned)ctas, a.kv_heads && a.rows == 1 ? 2 : 1), ROT_THREADS, smem,
           counted(stream)>>>(a);
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
