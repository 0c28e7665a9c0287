// Grouped attention on the fp32 pipes: fp32 inputs, and bf16 inputs that the
// tensor-core kernel does not take (widths that are no multiple of 8 or above
// 128, groups above 128, unaligned rows, negative scales).
//
// One CTA takes 32 rows of one K/V head (64 at widths above 128) and walks
// 64-key tiles; a thread holds 4 rows x 4 keys of the scores and 4 rows x DP/16
// columns of the output.  Four CTAs share an SM (two at widths above 64, one
// above 128): their barriers fall at different times, and their tiles fill the
// SMs where one tile of 128 rows and 512 threads left SMs idle (8 heads of 32, one
// prompt of 1001 tokens: 86 -> 45 us; 2 x 2048 tokens of 16/4 heads of 64: 675 ->
// 560 us; 16 rows 53 and 710 us, 2 rows a thread 60 and 800 us).  Both products
// read 16-byte vectors from shared memory (8 for 64 multiply-adds, 12 for 128 at
// DP = 128) into packed fp32x2 multiply-adds: the scores sum even and odd dimensions apart,
// so both factors are pairs as they lie.  Eight steps of either are unrolled, so
// that loads run ahead of the multiply-adds (5 to 9 % over 2 and 1).  The next K
// tile is fetched (cp.async) under the value product and the next V tile under
// the scores, in one buffer each.  The weights pass through shared memory between
// the 16 threads of a row.  Running maximum and sum, scores, weights and outputs
// are fp32.  Bound by the shared-memory reads that feed the multiply-adds, and in
// small calls by the chain of a tile: 2 x 2048 tokens of 32/8 heads of 128 take
// 2.01 ms, 34 TFLOP/s of the 74 of the fp32 pipes; 8 heads of 32, 2704 tokens in
// four prompts, 69 us.  bf16 rows are widened one element a load: 2 x 2048 tokens
// of 32/8 heads take 3.8 ms at width 128 (18 TFLOP/s) and 7.6 ms at 256.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "grouped_attention.cuh"

namespace grs {

constexpr int GA_KEYS = 64, GA_PS = GA_KEYS + 4;
constexpr int GA_I = 4;                                // rows of a thread

template <int DP>
struct GaShape {
  static constexpr int kRows = grouped_rows_tile(DP);
  static constexpr int kThreads = 16 * kRows / GA_I;   // 16 threads for GA_I rows
  static constexpr int kRowStep = kRows / GA_I;        // thread rows: rg + kRowStep i
  static constexpr int kQS = DP + 4;                   // padded row strides (floats)
  static constexpr int kSmem = (kRows * kQS + GA_KEYS * kQS + GA_KEYS * DP + kRows * GA_PS) * 4;
  static constexpr int kCtas = DP <= 64 ? 4 : DP <= 128 ? 2 : 1;   // of an SM
};

__device__ __forceinline__ void ga_copy16(float* dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(
                   (unsigned)__cvta_generic_to_shared(dst)),
               "l"(src), "r"(in ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void ga_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ga_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

// rows [t0, t0 + 64) of a K or V head into shared memory, zeros past `end` and
// past the width
template <typename T, int DP, int kStride, int kThreads, bool kAsync>
__device__ __forceinline__ void ga_load(float* dst, const T* src, int64_t st, int D, int t0,
                                        int end) {
  if constexpr (kAsync) {
#pragma unroll 4
    for (int i = threadIdx.x; i < GA_KEYS * DP / 4; i += kThreads) {
      const int t = i / (DP / 4), d = i % (DP / 4) * 4;
      const bool in = t0 + t < end && d < D;
      ga_copy16(dst + t * kStride + d, in ? src + (int64_t)(t0 + t) * st + d : src, in);
    }
  } else {
#pragma unroll 8
    for (int i = threadIdx.x; i < GA_KEYS * DP; i += kThreads) {
      const int t = i / DP, d = i % DP;
      dst[t * kStride + d] =
          t0 + t < end && d < D ? to_float(src[(int64_t)(t0 + t) * st + d]) : 0.f;
    }
  }
  ga_commit();
}

template <typename T, int DP, bool kCausal, bool kAsync>
__global__ void __launch_bounds__(GaShape<DP>::kThreads, GaShape<DP>::kCtas)
grouped_rows_kernel(const __grid_constant__ GroupedArgs<T> a) {
  using S = GaShape<DP>;
  extern __shared__ __align__(16) float ga_smem_raw[];
  float* qs = ga_smem_raw;                  // [kRows][kQS], scaled
  float* ks = qs + S::kRows * S::kQS;       // [GA_KEYS][kQS]
  float* vs = ks + GA_KEYS * S::kQS;        // [GA_KEYS][DP]
  float* ps = vs + GA_KEYS * DP;            // [kRows][GA_PS]
  // per row its keys; first and last key of any row, last first and first last
  __shared__ int row_begin[S::kRows], row_end[S::kRows], span[4];
  __shared__ int row_position[S::kRows], row_head[S::kRows];   // -1: no row
  constexpr int kPairs = DP / 32;           // output column pairs of a thread
  const int tid = threadIdx.x;
  const int rg = tid >> 4, cg = tid & 15;
  const int h = blockIdx.y;
  const int64_t total = (int64_t)a.positions * a.group;
  // the kernel that joins the slices may start as SMs fall free
  if (!kCausal) asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  // late rows of a causal tile see the most keys: they start first
  const int64_t row0 = (int64_t)(kCausal ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * S::kRows;

  if (tid == 0) {
    span[0] = span[3] = INT_MAX;
    span[1] = span[2] = 0;
  }
  __syncthreads();
  if (tid < S::kRows) {
    const int64_t r = row0 + tid;
    int begin = 0, end = 0, p = -1, head = 0;
    if (r < total) {
      p = (int)(r / a.group);
      head = h * a.group + (int)(r - (int64_t)p * a.group);
      if (kCausal) {
        causal_range(a.offsets, a.sequences, p, begin, end);
      } else {
        begin = min(a.keys, (int)blockIdx.z * a.slice_keys);
        end = min(a.keys, begin + a.slice_keys);
      }
    }
    row_begin[tid] = begin;
    row_end[tid] = end;
    row_position[tid] = p;
    row_head[tid] = head;
    if (end > begin) {
      atomicMin(&span[0], begin);
      atomicMax(&span[1], end);
      atomicMax(&span[2], begin);
      atomicMin(&span[3], end);
    }
  }
  __syncthreads();
  const int first = span[0], last = span[1], all_from = span[2], all_to = span[3];
  const T* kh = a.k + (int64_t)h * a.k_sh;
  const T* vh = a.v + (int64_t)h * a.v_sh;
  if (first < last) {
    ga_load<T, DP, S::kQS, S::kThreads, kAsync>(ks, kh, a.k_st, a.D, first, last);
    ga_load<T, DP, DP, S::kThreads, kAsync>(vs, vh, a.v_st, a.D, first, last);
  }
#pragma unroll 8
  for (int i = tid; i < S::kRows * DP; i += S::kThreads) {
    const int r = i / DP, d = i % DP, p = row_position[r];
    float x = 0.f;
    if (p >= 0 && d < a.D)
      x = to_float(a.q[(int64_t)p * a.q_sp + (int64_t)row_head[r] * a.q_sh + d]);
    qs[r * S::kQS + d] = x * a.scale_log2;
  }

  float2 acc[GA_I][kPairs];
  float m[GA_I], l[GA_I];
#pragma unroll
  for (int i = 0; i < GA_I; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) acc[i][j] = make_float2(0.f, 0.f);
  }

  for (int t0 = first; t0 < last; t0 += GA_KEYS) {
    ga_wait<1>();                           // K is here; V may be on its way
    __syncthreads();
    float s[GA_I][4];
    {
      float2 s2[GA_I][4];
#pragma unroll
      for (int i = 0; i < GA_I; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s2[i][j] = make_float2(0.f, 0.f);
#pragma unroll 8
      for (int d = 0; d < DP; d += 4) {
        float4 k4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          k4[j] = *reinterpret_cast<const float4*>(ks + (cg + 16 * j) * S::kQS + d);
#pragma unroll
        for (int i = 0; i < GA_I; ++i) {
          const float4 q4 = *reinterpret_cast<const float4*>(qs + (rg + S::kRowStep * i) * S::kQS + d);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s2[i][j] = __ffma2_rn(make_float2(q4.x, q4.y), make_float2(k4[j].x, k4[j].y), s2[i][j]);
            s2[i][j] = __ffma2_rn(make_float2(q4.z, q4.w), make_float2(k4[j].z, k4[j].w), s2[i][j]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < GA_I; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = s2[i][j].x + s2[i][j].y;
    }
    __syncthreads();                        // K is read
    ga_load<T, DP, S::kQS, S::kThreads, kAsync>(ks, kh, a.k_st, a.D, t0 + GA_KEYS, last);
    if (t0 < all_from || t0 + GA_KEYS > all_to) {
#pragma unroll
      for (int i = 0; i < GA_I; ++i) {
        const int from = row_begin[rg + S::kRowStep * i] - t0, to = row_end[rg + S::kRowStep * i] - t0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (cg + 16 * j < from || cg + 16 * j >= to) s[i][j] = -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < GA_I; ++i) {
      float top = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = fmaxf(top, m[i]);
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = exp2f(m[i] - base);
      m[i] = top;
      float sum = 0.f;
      float* p = ps + (rg + S::kRowStep * i) * GA_PS + cg;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = exp2f(s[i][j] - base);
        sum += w;
        p[16 * j] = w;
      }
      l[i] = l[i] * keep + sum;             // this thread's share of the row's sum
#pragma unroll
      for (int j = 0; j < kPairs; ++j)
        acc[i][j] = __fmul2_rn(acc[i][j], make_float2(keep, keep));
    }
    ga_wait<1>();                           // V is here
    __syncthreads();
#pragma unroll 8
    for (int t = 0; t < GA_KEYS; t += 4) {
      float4 p4[GA_I];
#pragma unroll
      for (int i = 0; i < GA_I; ++i)
        p4[i] = *reinterpret_cast<const float4*>(ps + (rg + S::kRowStep * i) * GA_PS + t);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float2 v2[kPairs];
        if constexpr (DP == 32) {
          v2[0] = *reinterpret_cast<const float2*>(vs + (t + k) * DP + 2 * cg);
        } else {
#pragma unroll
          for (int j = 0; j < kPairs / 2; ++j) {
            const float4 v4 = *reinterpret_cast<const float4*>(vs + (t + k) * DP + 64 * j + 4 * cg);
            v2[2 * j] = make_float2(v4.x, v4.y);
            v2[2 * j + 1] = make_float2(v4.z, v4.w);
          }
        }
#pragma unroll
        for (int i = 0; i < GA_I; ++i) {
          const float w = k == 0 ? p4[i].x : k == 1 ? p4[i].y : k == 2 ? p4[i].z : p4[i].w;
#pragma unroll
          for (int j = 0; j < kPairs; ++j) acc[i][j] = __ffma2_rn(make_float2(w, w), v2[j], acc[i][j]);
        }
      }
    }
    __syncthreads();                        // V is read
    ga_load<T, DP, DP, S::kThreads, kAsync>(vs, vh, a.v_st, a.D, t0 + GA_KEYS, last);
  }
  ga_wait<0>();

  unsigned again = 0;                       // rows (of GA_I) whose result is not finite
#pragma unroll
  for (int i = 0; i < GA_I; ++i) {
    float sum = l[i];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int r = rg + S::kRowStep * i, p = row_position[r], head = row_head[r];
    if (p < 0) continue;
    const bool seen = row_end[r] > row_begin[r];
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    bool odd = !(fabsf(sum) <= FLT_MAX);
#pragma unroll
    for (int j = 0; j < 2 * kPairs; ++j) {
      const int d = DP == 32 ? 2 * cg + j : 64 * (j / 4) + 4 * cg + (j & 3);
      const float x = (j & 1 ? acc[i][j / 2].y : acc[i][j / 2].x) * inv;
      if (d >= a.D) continue;
      if (kCausal) {
        if (seen || a.clear_rest)
          a.out[(int64_t)p * a.o_sp + (int64_t)head * a.o_sh + d] = from_float<T>(seen ? x : 0.f);
        odd |= !(fabsf(x) <= FLT_MAX);
      } else {
        a.part[(((int64_t)blockIdx.z * a.positions + p) * a.heads + head) * a.D + d] = x;
      }
    }
    if (!kCausal && cg == 0)
      a.part_lse[((int64_t)blockIdx.z * a.positions + p) * a.heads + head] =
          sum == 0.f ? -INFINITY : m[i] + log2f(sum);
    if (odd && seen) again |= 1u << i;
  }
  if constexpr (kCausal) {
    // the writes of the half warp's rows come first
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) again |= __shfl_xor_sync(0xffffffffu, again, o);
    __syncwarp();
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      unsigned todo = __shfl_sync(0xffffffffu, again, 16 * half);
      while (todo) {
        const int i = __ffs(todo) - 1;
        todo &= todo - 1;
        const int r = (tid >> 5) * 2 + half + S::kRowStep * i;
        causal_row_again<T, (DP + 31) / 32>(a, row_position[r], row_head[r], row_begin[r],
                                            row_end[r], 0, a.D);
      }
    }
  }
}

template <typename T, int DP, bool kCausal, bool kAsync>
static int rows_launch(const GroupedArgs<T>& a, cudaStream_t stream) {
  using S = GaShape<DP>;
  static_assert(S::kSmem + 4 * (4 * S::kRows + 4) <= 227 * 1024, "shared memory of a CTA");
  const int64_t tiles = ((int64_t)a.positions * a.group + S::kRows - 1) / S::kRows;
  if (tiles > INT_MAX || a.kv_heads > 65535 || (!kCausal && a.slices > 65535))
    return GRS_ERR_SHAPE;
  if (cudaFuncSetAttribute(grouped_rows_kernel<T, DP, kCausal, kAsync>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess)
    return GRS_ERR_CUDA;
  const dim3 grid((unsigned)tiles, a.kv_heads, kCausal ? 1 : a.slices);
  grouped_rows_kernel<T, DP, kCausal, kAsync>
      <<<grid, S::kThreads, S::kSmem, counted(stream)>>>(a);
  GRS_CUDA_CHECK_LAUNCH();
  return GRS_OK;
}

// 16-byte copies need rows of whole 16 bytes at 16-byte addresses
static bool rows_aligned(const GroupedArgs<float>& a) {
  return (reinterpret_cast<uintptr_t>(a.k) & 15) == 0 &&
         (reinterpret_cast<uintptr_t>(a.v) & 15) == 0 &&
         a.D % 4 == 0 && a.k_st % 4 == 0 && a.k_sh % 4 == 0 && a.v_st % 4 == 0 && a.v_sh % 4 == 0;
}

template <typename T, int DP>
static int rows_forms(const GroupedArgs<T>& a, cudaStream_t stream) {
  const bool causal = a.offsets != nullptr;
  if constexpr (sizeof(T) == 4)
    if (rows_aligned(a))
      return causal ? rows_launch<T, DP, true, true>(a, stream)
                    : rows_launch<T, DP, false, true>(a, stream);
  return causal ? rows_launch<T, DP, true, false>(a, stream)
                : rows_launch<T, DP, false, false>(a, stream);
}

template <typename T>
int grouped_rows_launch(const GroupedArgs<T>& a, cudaStream_t stream) {
  if (a.D <= 32) return rows_forms<T, 32>(a, stream);
  if (a.D <= 64) return rows_forms<T, 64>(a, stream);
  if (a.D <= 128) return rows_forms<T, 128>(a, stream);
  if (a.D <= 256) return rows_forms<T, 256>(a, stream);
  return GRS_ERR_SHAPE;
}

template int grouped_rows_launch<float>(const GroupedArgs<float>&, cudaStream_t);
template int grouped_rows_launch<__nv_bfloat16>(const GroupedArgs<__nv_bfloat16>&, cudaStream_t);

}  // namespace grs
