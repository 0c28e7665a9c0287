// Attention of query rows to keys shared by a group of heads: what the prompt
// and the shared-prefix entry points hand to the kernels.
//
// The rows of K/V head h are the pairs (position p, head h * group + g) in the
// order p * group + g, so one tile of rows reads its keys once for the whole
// group.  Two ranges of keys exist:
//   * causal: positions are tokens of packed sequences; position p of the
//     sequence that starts at s sees the keys s..p;
//   * slices: every row sees the keys [0, keys), cut into `slices` runs of
//     `slice_keys`; each slice leaves its normalised fp32 sum and the log2 of
//     its weight, which the reader joins.
#pragma once

#include "grs_common.cuh"

namespace grs {

constexpr float GA_LOG2E = 1.4426950408889634f;

template <typename T>
struct GroupedArgs {
  const T* q; int64_t q_sp, q_sh;          // [positions, heads, D], D contiguous
  const T* k; int64_t k_st, k_sh;          // [keys, kv_heads, D]
  const T* v; int64_t v_st, v_sh;
  int positions, keys, heads, kv_heads, group, D;
  float scale_log2;                        // softmax scale times log2(e)
  // causal
  const int32_t* offsets; int sequences;   // int32 [sequences + 1]
  T* out; int64_t o_sp, o_sh;              // [positions, heads, D]
  int clear_rest;                          // zero the rows outside every sequence
  // slices
  float* part;                             // fp32 [slices, positions, heads, D]
  float* part_lse;                         // fp32 [slices, positions, heads]
  int slices, slice_keys;
  int32_t* status;
};

// The keys [begin, end) of the sequence that position p belongs to, up to p
// itself; empty when p lies in no sequence.  Any offsets give a range inside
// [0, p]: what the array holds moves no access out of the tensors.
__device__ __forceinline__ void causal_range(const int32_t* __restrict__ offsets, int sequences,
                                             int p, int& begin, int& end) {
  int lo = 0, hi = sequences + 1;          // first j with offsets[j] > p
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(offsets + mid) <= p) lo = mid + 1; else hi = mid;
  }
  begin = end = 0;
  if (lo > 0 && lo <= sequences) {
    begin = min(max(__ldg(offsets + lo - 1), 0), p);
    end = p + 1;
  }
}

// One row of the causal form, by one warp, reading only the keys that the row
// sees.  The tiled kernels multiply masked keys by a weight of zero, which is
// nothing unless such a key's value is infinite or NaN (rows behind the last
// sequence, a neighbour sequence, a later token); rows whose tiled result is
// not finite are computed again here, columns [column0, column1) of at most
// 32 ND.
template <typename T, int ND>
__device__ __noinline__ void causal_row_again(const GroupedArgs<T>& a, int p, int head, int begin, int end,
                                              int column0, int column1) {
  const int lane = threadIdx.x & 31;
  const T* q = a.q + (int64_t)p * a.q_sp + (int64_t)head * a.q_sh;
  const T* kh = a.k + (int64_t)(head / a.group) * a.k_sh;
  const T* vh = a.v + (int64_t)(head / a.group) * a.v_sh;
  float m = -INFINITY, l = 0.f, acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = 0.f;
  for (int t0 = begin; t0 < end; t0 += 32) {
    const int t = t0 + lane;
    float s = -INFINITY;
    if (t < end) {
      const T* k = kh + (int64_t)t * a.k_st;
      float dot = 0.f;
#pragma unroll 1
      for (int d = 0; d < a.D; ++d) dot = fmaf(to_float(q[d]), to_float(k[d]), dot);
      s = dot * a.scale_log2;
    }
    const float top = fmaxf(m, warp_max(s));
    const float base = top == -INFINITY ? 0.f : top;
    const float w = exp2f(s - base);       // NaN scores stay NaN
    const float keep = exp2f(m - base);
    l = l * keep + warp_sum(w);
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] *= keep;
    m = top;
    const int n = min(32, end - t0);
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const T* v = vh + (int64_t)(t0 + j) * a.v_st;
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const int d = column0 + lane + 32 * i;
        if (d < column1) acc[i] = fmaf(wj, to_float(v[d]), acc[i]);
      }
    }
    // a NaN weight makes every later sum NaN: the row is decided
    if (l != l) break;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* o = a.out + (int64_t)p * a.o_sp + (int64_t)head * a.o_sh;
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int d = column0 + lane + 32 * i;
    if (d < column1) o[d] = from_float<T>(acc[i] * inv);
  }
}

// Rows of a tile of the rows kernel, by head width
constexpr int grouped_rows_tile(int width) { return width <= 128 ? 32 : 64; }

// Launchers; both return a grs_status.  The rows kernel takes every width up
// to 256, every group and any strides.
template <typename T> int grouped_rows_launch(const GroupedArgs<T>& a, cudaStream_t stream);

}  // namespace grs
