// Grouped attention on the fp32 pipes: fp32 inputs, and bf16 inputs that the
// tensor-core kernel does not take (widths that are no multiple of 8 or above
// 128, groups above 128, unaligned rows).
//
// One CTA of 128 threads takes 64 rows of one K/V head and walks 64-key tiles.
// Q, K and V stand in shared memory in fp32, Q and K transposed, so that a
// thread's 8 x 4 scores read three 16-byte vectors per dimension for 32
// multiply-adds; the weights go through shared memory (transposed) to the
// 8 x DP/16 outputs of the same half warp, four vectors per key for 64
// multiply-adds at DP = 128.  Running maximum and sum, scores and outputs are
// fp32.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "grouped_attention.cuh"

namespace grs {

constexpr int GA_ROWS = 64, GA_KEYS = 64, GA_THREADS = 128;
constexpr int GA_QS = GA_ROWS + 4, GA_KS = GA_KEYS + 4;   // transposed row strides (floats)

template <int DP>
constexpr int ga_smem() {
  return (DP * GA_QS + DP * GA_KS + GA_KEYS * DP + GA_KEYS * GA_QS) * 4;
}

template <typename T, int DP, bool kCausal>
__global__ void __launch_bounds__(GA_THREADS) grouped_rows_kernel(GroupedArgs<T> a) {
  extern __shared__ float ga_smem_raw[];
  float* qt = ga_smem_raw;                  // [DP][GA_QS]
  float* kt = qt + DP * GA_QS;              // [DP][GA_KS]
  float* vs = kt + DP * GA_KS;              // [GA_KEYS][DP]
  float* pt = vs + GA_KEYS * DP;            // [GA_KEYS][GA_QS]
  __shared__ int row_begin[GA_ROWS], row_end[GA_ROWS], span[2];
  constexpr int NV = DP / 16;               // output columns of a thread
  const int tid = threadIdx.x, lane = tid & 31;
  const int rg = tid >> 4, cg = tid & 15;   // 8 rows from 8 rg; keys and columns of cg
  const int h = blockIdx.y;
  const int64_t total = (int64_t)a.positions * a.group;
  // late rows of a causal tile see the most keys: they start first
  const int64_t row0 = (int64_t)(kCausal ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * GA_ROWS;

  if (tid < GA_ROWS) {
    const int64_t r = row0 + tid;
    int begin = 0, end = 0;
    if (r < total) {
      if (kCausal) {
        causal_range(a.offsets, a.sequences, (int)(r / a.group), begin, end);
      } else {
        begin = blockIdx.z * a.slice_keys;
        end = min(a.keys, begin + a.slice_keys);
      }
    }
    row_begin[tid] = begin;
    row_end[tid] = end;
  }
  if (tid == 0) { span[0] = INT_MAX; span[1] = 0; }
  __syncthreads();
  if (tid < GA_ROWS && row_end[tid] > row_begin[tid]) {
    atomicMin(&span[0], row_begin[tid]);
    atomicMax(&span[1], row_end[tid]);
  }
  for (int i = tid; i < GA_ROWS * DP; i += GA_THREADS) {
    const int r = i / DP, d = i % DP;
    const int64_t row = row0 + r;
    float x = 0.f;
    if (row < total && d < a.D)
      x = to_float(a.q[(row / a.group) * a.q_sp +
                       ((int64_t)h * a.group + row % a.group) * a.q_sh + d]);
    qt[d * GA_QS + r] = x * a.scale_log2;
  }
  __syncthreads();
  const int first = span[0], last = span[1];

  float acc[8][NV], m[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) acc[i][j] = 0.f;
  }
  int rb[8], re[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    rb[i] = row_begin[8 * rg + i];
    re[i] = row_end[8 * rg + i];
  }

  for (int t0 = first; t0 < last; t0 += GA_KEYS) {
    // keys along the lanes: the transposed writes hit every bank once
    for (int i = tid; i < GA_KEYS * DP; i += GA_THREADS) {
      const int t = i % GA_KEYS, d = i / GA_KEYS;
      float x = 0.f;
      if (t0 + t < last && d < a.D)
        x = to_float(a.k[(int64_t)(t0 + t) * a.k_st + (int64_t)h * a.k_sh + d]);
      kt[d * GA_KS + t] = x;
    }
    for (int i = tid; i < GA_KEYS * DP; i += GA_THREADS) {
      const int t = i / DP, d = i % DP;
      float x = 0.f;
      if (t0 + t < last && d < a.D)
        x = to_float(a.v[(int64_t)(t0 + t) * a.v_st + (int64_t)h * a.v_sh + d]);
      vs[i] = x;
    }
    __syncthreads();
    float s[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DP; ++d) {
      const float4 q0 = *reinterpret_cast<const float4*>(qt + d * GA_QS + 8 * rg);
      const float4 q1 = *reinterpret_cast<const float4*>(qt + d * GA_QS + 8 * rg + 4);
      const float4 k4 = *reinterpret_cast<const float4*>(kt + d * GA_KS + 4 * cg);
      const float qv[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
      const float kv[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = fmaf(qv[i], kv[j], s[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = t0 + 4 * cg + j;
        if (t < rb[i] || t >= re[i]) s[i][j] = -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = fmaxf(top, m[i]);
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = exp2f(m[i] - base);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(s[i][j] - base);
        sum += s[i][j];
      }
      l[i] = l[i] * keep + sum;             // this thread's share of the row's sum
      m[i] = top;
#pragma unroll
      for (int j = 0; j < NV; ++j) acc[i][j] *= keep;
    }
    // the weights of 8 rows pass between the 16 threads of the half warp
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float* p = pt + (4 * cg + j) * GA_QS + 8 * rg;
      *reinterpret_cast<float4*>(p) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(s[4][j], s[5][j], s[6][j], s[7][j]);
    }
    __syncwarp();
#pragma unroll 2
    for (int t = 0; t < GA_KEYS; ++t) {
      const float4 p0 = *reinterpret_cast<const float4*>(pt + t * GA_QS + 8 * rg);
      const float4 p1 = *reinterpret_cast<const float4*>(pt + t * GA_QS + 8 * rg + 4);
      const float pv[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
      float vv[NV];
      if constexpr (NV == 2) {
        const float2 v2 = *reinterpret_cast<const float2*>(vs + t * DP + 2 * cg);
        vv[0] = v2.x;
        vv[1] = v2.y;
      } else {
#pragma unroll
        for (int j = 0; j < NV / 4; ++j) {
          const float4 v4 = *reinterpret_cast<const float4*>(vs + t * DP + 64 * j + 4 * cg);
          vv[4 * j] = v4.x;
          vv[4 * j + 1] = v4.y;
          vv[4 * j + 2] = v4.z;
          vv[4 * j + 3] = v4.w;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < NV; ++j) acc[i][j] = fmaf(pv[i], vv[j], acc[i][j]);
    }
    __syncthreads();
  }

  unsigned again = 0;                       // rows (of 8) whose result is not finite
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float sum = l[i];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int64_t row = row0 + 8 * rg + i;
    if (row >= total) continue;
    const int p = (int)(row / a.group), head = h * a.group + (int)(row % a.group);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    bool odd = !(fabsf(sum) <= FLT_MAX);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = NV == 2 ? 2 * cg + j : 64 * (j / 4) + 4 * cg + (j & 3);
      const float x = acc[i][j] * inv;
      if (d >= a.D) continue;
      if (kCausal) {
        if (re[i] > rb[i] || a.clear_rest)
          a.out[(int64_t)p * a.o_sp + (int64_t)head * a.o_sh + d] = from_float<T>(x);
        odd |= !(fabsf(x) <= FLT_MAX);
      } else {
        a.part[(((int64_t)blockIdx.z * a.positions + p) * a.heads + head) * a.D + d] = x;
      }
    }
    if (!kCausal && cg == 0)
      a.part_lse[((int64_t)blockIdx.z * a.positions + p) * a.heads + head] =
          sum == 0.f ? -INFINITY : m[i] + log2f(sum);
    if (odd) again |= 1u << i;
  }
  if constexpr (kCausal) {
    // the whole warp holds rows 16 (warp) .. + 15; the writes above come first
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) again |= __shfl_xor_sync(0xffffffffu, again, o);
    __syncwarp();
    for (int half = 0; half < 2; ++half) {
      unsigned todo = __shfl_sync(0xffffffffu, again, 16 * half);
      while (todo) {
        const int i = __ffs(todo) - 1;
        todo &= todo - 1;
        const int r = (tid >> 5) * 16 + 8 * half + i;
        const int64_t row = row0 + r;
        if (row < total && row_end[r] > row_begin[r])
          causal_row_again<T, (DP + 31) / 32>(a, (int)(row / a.group),
                                              h * a.group + (int)(row % a.group), row_begin[r],
                                              row_end[r], 0, a.D);
      }
    }
  }
}

template <typename T, int DP, bool kCausal>
static int rows_launch(const GroupedArgs<T>& a, cudaStream_t stream) {
  const int64_t tiles = ((int64_t)a.positions * a.group + GA_ROWS - 1) / GA_ROWS;
  if (tiles > INT_MAX || a.kv_heads > 65535 || (!kCausal && a.slices > 65535))
    return GRS_ERR_SHAPE;
  if (cudaFuncSetAttribute(grouped_rows_kernel<T, DP, kCausal>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                           ga_smem<DP>()) != cudaSuccess)
    return GRS_ERR_CUDA;
  const dim3 grid((unsigned)tiles, a.kv_heads, kCausal ? 1 : a.slices);
  grouped_rows_kernel<T, DP, kCausal><<<grid, GA_THREADS, ga_smem<DP>(), counted(stream)>>>(a);
  GRS_CUDA_CHECK_LAUNCH();
  return GRS_OK;
}

template <typename T>
int grouped_rows_launch(const GroupedArgs<T>& a, cudaStream_t stream) {
  const bool causal = a.offsets != nullptr;
#define GRS_GA_WIDTH(DP)                                       \
  if (a.D <= DP)                                               \
    return causal ? rows_launch<T, DP, true>(a, stream) : rows_launch<T, DP, false>(a, stream)
  GRS_GA_WIDTH(32);
  GRS_GA_WIDTH(64);
  GRS_GA_WIDTH(128);
  GRS_GA_WIDTH(256);
#undef GRS_GA_WIDTH
  return GRS_ERR_SHAPE;
}

template int grouped_rows_launch<float>(const GroupedArgs<float>&, cudaStream_t);
template int grouped_rows_launch<__nv_bfloat16>(const GroupedArgs<__nv_bfloat16>&, cudaStream_t);

}  // namespace grs
