// One query per beam against a prefix that every beam shares and against the
// beam's own pages: grs_shared_prefix_attention.
//
// A long prefix is attention of beams * group rows per K/V head to the same
// keys, so its K/V are read once per tile of rows instead of once per beam; it
// is cut into slices when the tiles alone would leave SMs idle.  Each slice
// leaves its normalised fp32 sum and log2 weight in the workspace; the pages
// kernel adds the beam's own keys, joins all parts by their weights and writes
// the output.  A short prefix is read by the pages kernel itself.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "grouped_attention_tc.cuh"

namespace grs {

template <typename T>
struct PagesArgs {
  const T* q; int64_t q_sb, q_sh;
  // a short prefix that the pages' kernels read themselves, or 0 rows
  const T* pk; const T* pv; int64_t pk_st, pk_sh, pv_st, pv_sh; int prefix;
  const T* kc; const T* vc; int64_t kc_sp, kc_st, kc_sh;
  const int32_t* bt; int64_t bt_s; int max_blocks; const int32_t* lengths; int num_pages, page;
  const T* ck; const T* cv; int64_t ck_sb, ck_sh; const uint8_t* cvalid;
  const float* part; const float* part_lse; int slices;   // parts of the prefix
  float* page_part; float* page_lse;   // the same arrays, for page slices joined by a later kernel
  T* out; int64_t o_sb, o_sh;
  int batch, heads, kv_heads, group, D;
  float scale_log2;
  int32_t* status;
};

// The key and value rows of a beam's token t (K/V head h): prefix rows, then
// the first `past` tokens of its pages, then its current token; null where the
// page is not in the cache.
template <typename T>
__device__ __forceinline__ void pages_token(const PagesArgs<T>& a, int b, int h, int t, int past,
                                            const T*& k, const T*& v) {
  if (t < a.prefix) {
    k = a.pk + (int64_t)t * a.pk_st + (int64_t)h * a.pk_sh;
    v = a.pv + (int64_t)t * a.pv_st + (int64_t)h * a.pv_sh;
    return;
  }
  t -= a.prefix;
  int64_t at = (int64_t)b * a.ck_sb + (int64_t)h * a.ck_sh;
  if (t < past) {
    const int page = __ldg(a.bt + (int64_t)b * a.bt_s + t / a.page);
    if (page < 0 || page >= a.num_pages) {
      set_status(a.status, GRS_ERR_BAD_PAGE);
      k = v = nullptr;
      return;
    }
    at = (int64_t)page * a.kc_sp + (int64_t)(t % a.page) * a.kc_st + (int64_t)h * a.kc_sh;
  }
  k = (t < past ? a.kc : a.ck) + at;
  v = (t < past ? a.vc : a.cv) + at;
}

// fp32 pages, and bf16 layouts that the tensor-core form does not take.  One CTA
// of four warps per beam and kG heads of a K/V head, every warp taking each
// fourth run of 32 tokens: a lane per key for the scores (the key row in vectors
// of kVec elements against the queries in shared memory, up to 16 requested before
// the first is used), a lane per column for the values, 8 to 32 keys' rows in
// flight.  The warps take turns on the prefix slices too and meet in shared
// memory.  Bound by the latency of a run's loads, in large calls by the L1's rate
// for a lane per row: 200 beams of 500 tokens, 8/8 heads of 128, 154 us, 5.3 TB/s.
template <typename T, int DP, int kVec, int kG>
__global__ void __launch_bounds__(128) pages_rows_kernel(PagesArgs<T> a) {
  constexpr int ND = (DP + 31) / 32;
  constexpr int kSums = kG == 1 ? 4 : 1;    // running sums of a score
  constexpr int kFlight = DP <= 64 ? 32 : DP <= 128 ? 16 : 8;   // keys' value rows in flight
  constexpr unsigned kSome = 0xffffffffu >> (32 - kFlight);
  __shared__ __align__(16) float q[kG][DP];
  __shared__ float sums[4][kG][DP], tops[4][kG], totals[4][kG];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = (a.group + kG - 1) / kG;             // of a K/V head's group
  const int chunk = blockIdx.x % chunks, at = blockIdx.x / chunks;
  const int b = at / a.kv_heads, h = at % a.kv_heads;
  const int head0 = h * a.group + chunk * kG, heads = min(kG, a.group - chunk * kG);
#pragma unroll
  for (int g = 0; g < kG; ++g)
    for (int d = threadIdx.x; d < DP; d += 128)
      q[g][d] = g < heads && d < a.D
                    ? to_float(a.q[(int64_t)b * a.q_sb + (int64_t)(head0 + g) * a.q_sh + d]) *
                          a.scale_log2
                    : 0.f;

  const int room = a.max_blocks * a.page;
  int past = a.lengths ? a.lengths[b] : 0;
  if (past < 0 || past > room) {
    if (threadIdx.x == 0) set_status(a.status, GRS_ERR_LENGTH);
    past = min(max(past, 0), room);
  }
  const bool cur = a.ck != nullptr && (a.cvalid == nullptr || a.cvalid[b] != 0);
  const int total = a.prefix + past + (cur ? 1 : 0);
  __syncthreads();

  float m[kG], l[kG], acc[kG][ND];          // l: this lane's keys
#pragma unroll
  for (int g = 0; g < kG; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[g][i] = 0.f;
  }
  for (int t0 = 32 * warp; t0 < total; t0 += 128) {
    const int t = t0 + lane;
    const T *k = nullptr, *v = nullptr;
    if (t < total) pages_token(a, b, h, t, past, k, v);
    const unsigned valid = __ballot_sync(0xffffffffu, k != nullptr);
    float w[kG];                            // scores, then weights
#pragma unroll
    for (int g = 0; g < kG; ++g) w[g] = -INFINITY;
    if (k) {
      float dot[kG][kSums];
#pragma unroll
      for (int g = 0; g < kG; ++g)
#pragma unroll
        for (int j = 0; j < kSums; ++j) dot[g][j] = 0.f;
      if constexpr (kVec > 1) {
        constexpr int kAhead = DP / kVec < 16 ? DP / kVec : 16;   // vectors in flight
#pragma unroll
        for (int d0 = 0; d0 < DP; d0 += kAhead * kVec) {
          uint4 y[kAhead];
#pragma unroll
          for (int n = 0; n < kAhead; ++n) {
            y[n] = make_uint4(0, 0, 0, 0);
            if (d0 + n * kVec < a.D) y[n] = __ldg(reinterpret_cast<const uint4*>(k + d0 + n * kVec));
          }
#pragma unroll
          for (int n = 0; n < kAhead; ++n) {
            const uint32_t words[4] = {y[n].x, y[n].y, y[n].z, y[n].w};
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
              const float x = kVec == 4 ? __uint_as_float(words[j])
                                        : __uint_as_float(j & 1 ? words[j / 2] & 0xffff0000u
                                                                : words[j / 2] << 16);
              const int d = d0 + n * kVec + j;
#pragma unroll
              for (int g = 0; g < kG; ++g)
                dot[g][d % kSums] = fmaf(q[g][d], x, dot[g][d % kSums]);
            }
          }
        }
      } else {
#pragma unroll 8
        for (int d = 0; d < a.D; ++d) {
          const float x = to_float(k[d]);
#pragma unroll
          for (int g = 0; g < kG; ++g) dot[g][0] = fmaf(q[g][d], x, dot[g][0]);
        }
      }
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        w[g] = dot[g][0];
        if constexpr (kSums == 4) w[g] = (w[g] + dot[g][1]) + (dot[g][2] + dot[g][3]);
      }
    }
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      const float top = fmaxf(m[g], warp_max(w[g]));
      const float base = top == -INFINITY ? 0.f : top;
      w[g] = exp2f(w[g] - base);
      const float keep = exp2f(m[g] - base);
      l[g] = l[g] * keep + w[g];
#pragma unroll
      for (int i = 0; i < ND; ++i) acc[g][i] *= keep;
      m[g] = top;
    }
#pragma unroll
    for (int j0 = 0; j0 < 32; j0 += kFlight) {
      if (((valid >> j0) & kSome) == 0) continue;
      float x[kFlight][ND];
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const T* vj = reinterpret_cast<const T*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v), j0 + j));
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          const int d = lane + 32 * i;
          x[j][i] = ((valid >> (j0 + j)) & 1) && d < a.D ? to_float(vj[d]) : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < kFlight; ++j)
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          const float wj = __shfl_sync(0xffffffffu, w[g], j0 + j);
#pragma unroll
          for (int i = 0; i < ND; ++i) acc[g][i] = fmaf(wj, x[j][i], acc[g][i]);
        }
    }
  }

  // join: weights exp2(lse_i - max lse); the pages' sums enter unnormalised
  asm volatile("griddepcontrol.wait;\n" ::: "memory");   // the prefix slices are written
  const int64_t stride = (int64_t)a.batch * a.heads, row0 = (int64_t)b * a.heads + head0;
#pragma unroll
  for (int g = 0; g < kG; ++g)
    if (lane == 0) tops[warp][g] = m[g];
  __syncthreads();
#pragma unroll
  for (int g = 0; g < kG; ++g) {
    const int64_t row = row0 + g;
    const int slices = g < heads ? a.slices : 0;
    float top = fmaxf(fmaxf(tops[0][g], tops[1][g]), fmaxf(tops[2][g], tops[3][g]));
    for (int i = lane; i < slices; i += 32) top = fmaxf(top, a.part_lse[i * stride + row]);
    top = warp_max(top);
    const float base = top == -INFINITY ? 0.f : top;
    const float own = exp2f(m[g] - base);
    float norm = warp_sum(l[g]) * own;
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[g][i] *= own;
    for (int p0 = warp; p0 < slices; p0 += 16) {
      float w[4], x[4][ND];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = p0 + 4 * j;
        w[j] = i < slices ? a.part_lse[i * stride + row] : -INFINITY;
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const int d = lane + 32 * n;
          x[j][n] = i < slices && d < a.D ? a.part[(i * stride + row) * a.D + d] : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2f(w[j] - base);
        norm += e;
#pragma unroll
        for (int n = 0; n < ND; ++n) acc[g][n] = fmaf(e, x[j][n], acc[g][n]);
      }
    }
#pragma unroll
    for (int i = 0; i < ND; ++i)
      if (lane + 32 * i < DP) sums[warp][g][lane + 32 * i] = acc[g][i];
    if (lane == 0) totals[warp][g] = norm;
  }
  __syncthreads();
#pragma unroll
  for (int g = 0; g < kG; ++g) {
    if (g >= heads) break;
    const float norm = (totals[0][g] + totals[1][g]) + (totals[2][g] + totals[3][g]);
    const float inv = norm == 0.f ? 0.f : 1.f / norm;
    T* o = a.out + (int64_t)b * a.o_sb + (int64_t)(head0 + g) * a.o_sh;
    for (int d = threadIdx.x; d < a.D; d += 128)
      o[d] = from_float<T>(
          ((sums[0][g][d] + sums[1][g][d]) + (sums[2][g][d] + sums[3][g][d])) * inv);
  }
}

// Whether a CTA takes four heads of a group: their keys and values are read
// once, unless single heads fit the SMs (fp32, 32/8 heads of 128: 200 beams of
// 500 tokens 503 -> 207 us, 4.0 TB/s, 32 of 64 17 -> 10; 4 of 1000 44 against 50;
// 16/8 heads, 200 of 500 269 -> 205, 4 of 1000 44 against 50).
template <typename T>
static bool pages_rows_few(const PagesArgs<T>& p) {
  return p.group > 1 && (int64_t)p.batch * p.heads > 148;
}

template <typename T>
static int pages_rows_launch(const PagesArgs<T>& p, bool after_prefix, cudaStream_t stream) {
  const bool few = pages_rows_few(p);
  const int64_t ctas = (int64_t)p.batch * p.kv_heads * (few ? (p.group + 3) / 4 : p.group);
  if (ctas > INT_MAX) return GRS_ERR_SHAPE;
  constexpr int kVec = 16 / sizeof(T);
  const auto whole = [](const void* at) { return (reinterpret_cast<uintptr_t>(at) & 15) == 0; };
  const bool prefix_vec =
      p.prefix == 0 || (whole(p.pk) && p.pk_st % kVec == 0 && p.pk_sh % kVec == 0);
  const bool vec = p.D % kVec == 0 && prefix_vec && whole(p.kc) && whole(p.ck) &&
                   p.kc_sp % kVec == 0 && p.kc_st % kVec == 0 && p.kc_sh % kVec == 0 &&
                   p.ck_sb % kVec == 0 && p.ck_sh % kVec == 0;
  // starts under the prefix kernel's tail; its join waits for the slices
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)ctas);
  config.blockDim = dim3(128);
  config.stream = counted(stream);
  config.attrs = &attr;
  config.numAttrs = after_prefix ? 1 : 0;
  const auto go = [&](auto width) {
    constexpr int DP = decltype(width)::value;
    if (few)
      return vec ? cudaLaunchKernelEx(&config, pages_rows_kernel<T, DP, kVec, 4>, p)
                 : cudaLaunchKernelEx(&config, pages_rows_kernel<T, DP, 1, 4>, p);
    return vec ? cudaLaunchKernelEx(&config, pages_rows_kernel<T, DP, kVec, 1>, p)
               : cudaLaunchKernelEx(&config, pages_rows_kernel<T, DP, 1, 1>, p);
  };
  const cudaError_t status = p.D <= 32    ? go(std::integral_constant<int, 32>{})
                             : p.D <= 64  ? go(std::integral_constant<int, 64>{})
                             : p.D <= 128 ? go(std::integral_constant<int, 128>{})
                                          : go(std::integral_constant<int, 256>{});
  if (status != cudaSuccess) return GRS_ERR_CUDA;
  GRS_CUDA_CHECK_LAUNCH();
  return GRS_OK;
}

// ---- bf16 pages on the tensor cores -------------------------------------------
// One CTA of `warps` warps per (beam, K/V head, 16 query heads), each warp
// taking every warps-th run of 32 tokens.  The pages are read once and nothing
// else is large, so memory bounds it: every lane fetches 16-byte pieces of the
// rows straight into mma.m16n8k16 operands, without shared memory.  A product
// does not care in which order its inner dimension is summed, so lane t of a
// quad takes the pieces t, t + 4, ... of a key row for its K fragments (the
// query fragments are loaded in the same order), and for V the lane's column
// index picks the piece and the eight elements of a piece go to eight
// different tiles; two keys' pieces are interleaved by byte permutes.  Groups
// of more than 8 heads take the heads as the 16 rows of both products (the
// weights leave the first in the layout of the second's A operand); groups of
// up to 8 (kFew) take keys, then value columns as rows and the heads as the 8
// columns, with two 8 x 8 transposes of the weights in between: half the
// instructions, accumulators and query registers.  The warps' sums meet in
// shared memory and are joined there with the prefix slices; only that join
// waits for the prefix kernel.  256 beams of 1024 tokens in pages of 16, 32/8
// heads of 128, take 190 us: 5.66 TB/s, 0.87 of the measured copy (267 us with
// the heads as rows).
constexpr int PG_HEADS = 16;

__device__ __forceinline__ void pg_mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float pg_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pg_pack(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <int DP>
struct PgShape {
  static constexpr int kPiece = DP >= 64 ? 8 : 4;         // V elements of a lane's piece
  static constexpr int kRuns = DP / (8 * kPiece);         // pieces of a lane
  static constexpr int kKey = DP / 32;                    // 16-byte K pieces of a lane
  static constexpr int kStride = DP + 4;                  // row of the joined sums (floats)
};

__device__ __forceinline__ uint32_t pg_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

// x += the parts first, first + step, ... of one (beam, head), four columns a
// lane, by their weights against `base`; returns the weights' sum.  The weights
// of 32 parts are taken at once, a lane each, so that the rows' loads depend on
// nothing and go out together.
__device__ __forceinline__ float pg_add_parts(const PagesArgs<__nv_bfloat16>& a, int parts,
                                              int first, int step, int64_t at, float base,
                                              float4& x) {
  const int lane = threadIdx.x & 31, d = 4 * lane;
  const int64_t stride = (int64_t)a.batch * a.heads;
  float norm = 0.f;
  for (int p0 = first; p0 < parts; p0 += 32 * step) {
    const int mine = p0 + lane * step;
    const float w = mine < parts ? pg_exp2(a.part_lse[mine * stride + at] - base) : 0.f;
    norm += warp_sum(w);
    const int n = min(32, (parts - p0 + step - 1) / step);
    for (int i0 = 0; i0 < n; i0 += 8) {
      float4 y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i0 + i < n && d < a.D)
          y[i] = *reinterpret_cast<const float4*>(
              a.part + ((p0 + (i0 + i) * step) * stride + at) * a.D + d);
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
  return norm;
}

template <int DP, bool kFew>
__global__ void __launch_bounds__(256) pages_mma_kernel(PagesArgs<__nv_bfloat16> a) {
  using S = PgShape<DP>;
  using T = __nv_bfloat16;
  extern __shared__ float pg_smem[];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int chunks = (a.group + PG_HEADS - 1) / PG_HEADS;
  const int b = blockIdx.x / (a.kv_heads * chunks);
  const int h = blockIdx.x / chunks % a.kv_heads;
  const int head0 = h * a.group + blockIdx.x % chunks * PG_HEADS;
  const int n_heads = min(PG_HEADS, (h + 1) * a.group - head0);

  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  constexpr int rows = kFew ? 8 : PG_HEADS;
  // query fragments: heads g and g + 8 (or g alone), pieces t, t + 4, ...
  uint32_t qa[2 * S::kKey][kFew ? 2 : 4];
#pragma unroll
  for (int i = 0; i < S::kKey; ++i) {
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    const int d = 8 * (t + 4 * i);
    const T* q = a.q + (int64_t)b * a.q_sb + (int64_t)(head0 + g) * a.q_sh + d;
    if (d < a.D && g < n_heads) lo = *reinterpret_cast<const uint4*>(q);
    if constexpr (kFew) {
      qa[2 * i][0] = lo.x;
      qa[2 * i][1] = lo.y;
      qa[2 * i + 1][0] = lo.z;
      qa[2 * i + 1][1] = lo.w;
    } else {
      if (d < a.D && g + 8 < n_heads) hi = *reinterpret_cast<const uint4*>(q + 8 * a.q_sh);
      qa[2 * i][0] = lo.x;
      qa[2 * i][1] = hi.x;
      qa[2 * i][2] = lo.y;
      qa[2 * i][3] = hi.y;
      qa[2 * i + 1][0] = lo.z;
      qa[2 * i + 1][1] = hi.z;
      qa[2 * i + 1][2] = lo.w;
      qa[2 * i + 1][3] = hi.w;
    }
  }

  const int room = a.max_blocks * a.page;
  int past = a.lengths ? a.lengths[b] : 0;
  if (past < 0 || past > room) {
    if (threadIdx.x == 0) set_status(a.status, GRS_ERR_LENGTH);
    past = min(max(past, 0), room);
  }
  const bool cur = a.ck != nullptr && (a.cvalid == nullptr || a.cvalid[b] != 0);
  const int total = a.prefix + past + (cur ? 1 : 0);
  const int runs = (total + 31) / 32;
  const int run_lo = (int)((int64_t)runs * blockIdx.y / gridDim.y);
  const int run_hi = (int)((int64_t)runs * (blockIdx.y + 1) / gridDim.y);
  const auto place = [&](int run, const T*& k, const T*& v) {   // rows of token 32 run + lane
    const int tok = run * 32 + lane;
    k = v = nullptr;
    if (run < run_hi && tok < total) pages_token(a, b, h, tok, past, k, v);
  };

  // kFew: columns (d, d + 1) x heads (2t, 2t + 1), d = piece (g + 8 j) + 2 i;
  // else: heads (g, g + 8) x columns of the pieces 2t and 2t + 1
  constexpr int kTiles = kFew ? DP / 16 : DP / 8;
  float acc[kTiles][4];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const T *next_k, *next_v;
  place(run_lo + warp, next_k, next_v);
  for (int run = run_lo + warp; run < run_hi; run += warps) {
    const unsigned valid = __ballot_sync(0xffffffffu, next_k != nullptr);
    const unsigned long long k_at = reinterpret_cast<unsigned long long>(next_k);
    const unsigned long long v_at = reinterpret_cast<unsigned long long>(next_v);
    place(run + warps, next_k, next_v);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (((valid >> (16 * half)) & 0xffffu) == 0) continue;
      uint4 kr[2][S::kKey];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const T* k = reinterpret_cast<const T*>(
            __shfl_sync(0xffffffffu, k_at, 16 * half + 8 * n + g));
#pragma unroll
        for (int i = 0; i < S::kKey; ++i) {
          const int d = 8 * (t + 4 * i);
          kr[n][i] = make_uint4(0, 0, 0, 0);
          if (k && d < a.D) kr[n][i] = __ldg(reinterpret_cast<const uint4*>(k + d));
        }
      }
      // values of keys 2t, 2t + 1, 2t + 8, 2t + 9
      uint32_t vr[4][S::kRuns][S::kPiece / 2];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int j = 16 * half + 2 * t + (n & 1) + 8 * (n >> 1);
        const T* v = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, v_at, j));
#pragma unroll
        for (int i = 0; i < S::kRuns; ++i) {
          const int d = S::kPiece * (g + 8 * i);
          if constexpr (S::kPiece == 8) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (v && d < a.D) w = __ldg(reinterpret_cast<const uint4*>(v + d));
            vr[n][i][0] = w.x;
            vr[n][i][1] = w.y;
            vr[n][i][2] = w.z;
            vr[n][i][3] = w.w;
          } else {
            uint2 w = make_uint2(0, 0);
            if (v && d < a.D) w = __ldg(reinterpret_cast<const uint2*>(v + d));
            vr[n][i][0] = w.x;
            vr[n][i][1] = w.y;
          }
        }
      }
      if constexpr (kFew) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};   // keys (g, g + 8) x heads (2t, 2t + 1)
#pragma unroll
        for (int i = 0; i < S::kKey; ++i) {
          const uint32_t k0[4] = {kr[0][i].x, kr[1][i].x, kr[0][i].y, kr[1][i].y};
          const uint32_t k1[4] = {kr[0][i].z, kr[1][i].z, kr[0][i].w, kr[1][i].w};
          pg_mma(s, k0, qa[2 * i][0], qa[2 * i][1]);
          pg_mma(s, k1, qa[2 * i + 1][0], qa[2 * i + 1][1]);
        }
        bool grown = false;
        float top[2];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const bool ok = (valid >> (16 * half + g + 8 * (c >> 1))) & 1;
          s[c] = ok ? s[c] * a.scale_log2 : -INFINITY;
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          top[r] = fmaxf(s[r], s[r + 2]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1)
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], o));
          grown |= top[r] > m[r];
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float now = fmaxf(m[r], top[r]);
            const float keep = now == -INFINITY ? 1.f : pg_exp2(m[r] - now);
            m[r] = now;
            l[r] *= keep;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
              acc[i][r] *= keep;
              acc[i][r + 2] *= keep;
            }
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[c] = pg_exp2(s[c] - (m[c & 1] == -INFINITY ? 0.f : m[c & 1]));
          l[c & 1] += s[c];
        }
        const uint32_t p0 = pg_transpose(pg_pack(s[0], s[1]));
        const uint32_t p1 = pg_transpose(pg_pack(s[2], s[3]));
#pragma unroll
        for (int i = 0; i < S::kRuns; ++i)
#pragma unroll
          for (int e = 0; e < S::kPiece / 2; ++e) {
            const uint32_t va[4] = {__byte_perm(vr[0][i][e], vr[1][i][e], 0x5410u),
                                    __byte_perm(vr[0][i][e], vr[1][i][e], 0x7632u),
                                    __byte_perm(vr[2][i][e], vr[3][i][e], 0x5410u),
                                    __byte_perm(vr[2][i][e], vr[3][i][e], 0x7632u)};
            pg_mma(acc[i * (S::kPiece / 2) + e], va, p0, p1);
          }
      } else {
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
          for (int i = 0; i < S::kKey; ++i) {
            pg_mma(s[n], qa[2 * i], kr[n][i].x, kr[n][i].y);
            pg_mma(s[n], qa[2 * i + 1], kr[n][i].z, kr[n][i].w);
          }
        }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const bool ok = (valid >> (16 * half + 8 * n + 2 * t + (c & 1))) & 1;
            s[n][c] = ok ? s[n][c] * a.scale_log2 : -INFINITY;
            top[c >> 1] = fmaxf(top[c >> 1], s[n][c]);
          }
        float base[2];
        bool grown = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
          grown |= top[r] > m[r];
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float now = fmaxf(m[r], top[r]);
            const float keep = now == -INFINITY ? 1.f : pg_exp2(m[r] - now);
            m[r] = now;
            l[r] *= keep;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
              acc[i][2 * r] *= keep;
              acc[i][2 * r + 1] *= keep;
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) base[r] = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[n][c] = pg_exp2(s[n][c] - base[c >> 1]);
            l[c >> 1] += s[n][c];
          }
        const uint32_t pa[4] = {pg_pack(s[0][0], s[0][1]), pg_pack(s[0][2], s[0][3]),
                                pg_pack(s[1][0], s[1][1]), pg_pack(s[1][2], s[1][3])};
#pragma unroll
        for (int i = 0; i < S::kRuns; ++i)
#pragma unroll
          for (int e = 0; e < S::kPiece; ++e) {
            const unsigned pick = (e & 1) ? 0x7632u : 0x5410u;
            pg_mma(acc[i * S::kPiece + e], pa,
                   __byte_perm(vr[0][i][e >> 1], vr[1][i][e >> 1], pick),
                   __byte_perm(vr[2][i][e >> 1], vr[3][i][e >> 1], pick));
          }
      }
    }
  }

  // each warp's state into shared memory
  float* sums = pg_smem;                                   // [warps][rows][kStride]
  float* tops = sums + warps * rows * S::kStride;
  float* totals = tops + warps * rows;
  if constexpr (kFew) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
      const int head = 2 * t + r;
      float* row = sums + (warp * rows + head) * S::kStride;
#pragma unroll
      for (int i = 0; i < S::kRuns; ++i)
#pragma unroll
        for (int e = 0; e < S::kPiece; e += 4) {
          const int at = i * (S::kPiece / 2) + e / 2;
          *reinterpret_cast<float4*>(row + S::kPiece * (g + 8 * i) + e) =
              make_float4(acc[at][r], acc[at][r + 2], acc[at + 1][r], acc[at + 1][r + 2]);
        }
      if (g == 0) {
        tops[warp * rows + head] = m[r];
        totals[warp * rows + head] = l[r];
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      const int head = g + 8 * r;
      float* row = sums + (warp * rows + head) * S::kStride;
#pragma unroll
      for (int i = 0; i < S::kRuns; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < S::kPiece; e += 4)
            *reinterpret_cast<float4*>(row + S::kPiece * (2 * t + c + 8 * i) + e) = make_float4(
                acc[i * S::kPiece + e][2 * r + c], acc[i * S::kPiece + e + 1][2 * r + c],
                acc[i * S::kPiece + e + 2][2 * r + c], acc[i * S::kPiece + e + 3][2 * r + c]);
      if (t == 0) {
        tops[warp * rows + head] = m[r];
        totals[warp * rows + head] = l[r];
      }
    }
  }
  __syncthreads();
  // The prefix slices are written.  Where a later kernel joins, one CTA waits
  // for all, so that this kernel ends behind the prefix kernel, and the others
  // leave their SMs to the CTAs still to come.
  const bool last = a.page_part == nullptr;
  if (last || (blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1))
    asm volatile("griddepcontrol.wait;\n" ::: "memory");

  // The warps' sums and the prefix slices are joined by a warp per head, or by
  // several that take turns on the parts; lane = 4 columns.
  const int64_t stride = (int64_t)a.batch * a.heads;
  const int parts = last ? a.slices : 0, teams = max(1, warps / n_heads);
  const int team = teams > 1 ? warp / n_heads : 0, d = 4 * lane;
  float4* shared_x = reinterpret_cast<float4*>(totals + warps * rows);   // [warps][32]
  float* shared_norm = reinterpret_cast<float*>(shared_x + warps * 32);
  const auto finish = [&](int head, float4 x, float norm, float base) {
    const int64_t at = (int64_t)b * a.heads + head0 + head;
    const float inv = norm == 0.f ? 0.f : 1.f / norm;
    x = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    if (last) {
      if (d < a.D)
        *reinterpret_cast<uint2*>(a.out + (int64_t)b * a.o_sb + (int64_t)(head0 + head) * a.o_sh +
                                  d) = make_uint2(pg_pack(x.x, x.y), pg_pack(x.z, x.w));
    } else {
      const int64_t to = (a.slices + blockIdx.y) * stride + at;
      if (d < a.D) *reinterpret_cast<float4*>(a.page_part + to * a.D + d) = x;
      if (lane == 0) a.page_lse[to] = norm == 0.f ? -INFINITY : base + log2f(norm);
    }
  };
  for (int head = teams > 1 ? warp % n_heads : warp; head < n_heads && team < teams;
       head += teams > 1 ? n_heads : warps) {
    const int64_t at = (int64_t)b * a.heads + head0 + head;
    float top = -INFINITY;
    for (int i = lane; i < warps; i += 32) top = fmaxf(top, tops[i * rows + head]);
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, a.part_lse[i * stride + at]);
    top = warp_max(top);
    const float base = top == -INFINITY ? 0.f : top;
    float norm = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = team; i < warps; i += teams) {
      const float w = pg_exp2(tops[i * rows + head] - base);
      norm = fmaf(w, totals[i * rows + head], norm);
      if (d < DP) {
        const float4 y = *reinterpret_cast<const float4*>(sums + (i * rows + head) * S::kStride + d);
        x.x = fmaf(w, y.x, x.x);
        x.y = fmaf(w, y.y, x.y);
        x.z = fmaf(w, y.z, x.z);
        x.w = fmaf(w, y.w, x.w);
      }
    }
    norm += pg_add_parts(a, parts, team, teams, at, base, x);
    if (teams == 1) {
      finish(head, x, norm, base);
    } else {
      shared_x[warp * 32 + lane] = x;
      if (lane == 0) shared_norm[2 * warp] = norm, shared_norm[2 * warp + 1] = base;
    }
  }
  if (teams > 1) {
    __syncthreads();
    if (warp < n_heads) {
      float4 x = shared_x[warp * 32 + lane];
      float norm = shared_norm[2 * warp];
      for (int i = 1; i < teams; ++i) {
        const float4 y = shared_x[(warp + i * n_heads) * 32 + lane];
        x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        norm += shared_norm[2 * (warp + i * n_heads)];
      }
      finish(warp, x, norm, shared_norm[2 * warp + 1]);
    }
  }
}

// The join alone: `team` (1 or 4) of a CTA's four warps per (beam, head).
__global__ void __launch_bounds__(128) join_parts_kernel(PagesArgs<__nv_bfloat16> a, int parts,
                                                         int team) {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");   // launched under the pages kernel
  __shared__ float4 xs[4][32];
  __shared__ float norms[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t stride = (int64_t)a.batch * a.heads;
  const int64_t at = team == 4 ? blockIdx.x : (int64_t)blockIdx.x * 4 + warp;
  if (at >= stride) return;                // whole CTAs, or warps that meet nobody
  float top = -INFINITY;
  for (int i = lane; i < parts; i += 32) top = fmaxf(top, a.part_lse[i * stride + at]);
  top = warp_max(top);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float norm = pg_add_parts(a, parts, team == 4 ? warp : 0, team, at,
                            top == -INFINITY ? 0.f : top, x);
  if (team == 4) {
    xs[warp][lane] = x;
    if (lane == 0) norms[warp] = norm;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      const float4 y = xs[i][lane];
      x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
      norm += norms[i];
    }
  }
  const float inv = norm == 0.f ? 0.f : 1.f / norm;
  const int d = 4 * lane;
  if (d < a.D)
    *reinterpret_cast<uint2*>(a.out + at / a.heads * a.o_sb + at % a.heads * a.o_sh + d) =
        make_uint2(pg_pack(x.x * inv, x.y * inv), pg_pack(x.z * inv, x.w * inv));
}

// How the prefix is cut: `parts` partial sums, `keys` per slice (two parts per
// slice when the tensor-core kernel's slots halve it).
struct PrefixPlan {
  int slices, parts, keys;
};

// fp32 rows: the count that gives the SM with most CTAs the least work, a CTA
// paying about one 64-key block for its start and end (64 beams of 32/8 heads of
// 128 over 4000 keys: 192 / 320 / 448 / 576 / 832 CTAs took 224 / 209 / 204 / 174
// / 190 us, 16 beams 144 / 256 / 336 / 512 CTAs 68 / 68 / 81 / 78 us).  Measured
// up to width 128; above, where an SM holds one CTA, it is taken as it is.
static PrefixPlan rows_plan(int batch, int group, int kv_heads, int D, int keys) {
  if (keys <= 0) return {0, 0, 0};
  const int64_t rows = grouped_rows_tile(D);
  const int64_t tiles = ((int64_t)batch * group + rows - 1) / rows * kv_heads;
  const int blocks = (keys + 63) / 64, most = std::min(64, blocks);
  const int64_t least = (tiles + 147) / 148;
  int64_t best = INT64_MAX;
  int slices = 1, each = blocks;
  for (int64_t ctas = least; ctas < least + 8; ++ctas) {   // of an SM
    // as many slices as this allows, then as few as give the same length
    const int z = (int)std::min<int64_t>(148 * ctas / tiles, most);
    const int length = (blocks + z - 1) / z;
    if (ctas * (length + 1) < best) {
      best = ctas * (length + 1);
      each = length;
      slices = (blocks + length - 1) / length;
    }
    if (z == most) break;
  }
  return {slices, slices, each * 64};
}

// Tensor cores: the count whose waves of 148 CTAs take the fewest 128-key
// blocks, each wave paying about four blocks for its start and end and every
// part the write and read of its fp32 sums, mostly in L2 (a block takes about
// 1.1 us; measured at width 128 and taken for the narrower ones too).
static PrefixPlan tc_plan(int batch, int heads, int kv_heads, int D, int keys) {
  if (keys <= 0) return {0, 0, 0};
  const int group = heads / kv_heads;
  const bool split = grouped_tc_split(batch, group);
  const int pps = std::max(1, 128 / group) * (split ? 1 : 2);
  const int64_t tiles = ((int64_t)batch + pps - 1) / pps * kv_heads;
  // slots of a split slice take turns on half the blocks each
  const int blocks = (keys + 127) / 128, per = split ? 2 : 1;
  const double join = 3.0 * batch * heads * D / 6.5e12 / 1.1e-6 + 0.02;
  const int most = std::min(64, (blocks + per - 1) / per);
  const int64_t least_waves = (tiles + 147) / 148;
  double best = 1e30;
  int slices = 1;
  for (int64_t waves = least_waves; waves < least_waves + 8; ++waves) {
    // as many slices as these waves hold, then as few as give the same length
    int z = (int)std::min<int64_t>(148 * waves / tiles, most);
    const int each = ((blocks + z - 1) / z + per - 1) / per;
    const double cost = (double)waves * (each + 4) + join * per * ((blocks + each * per - 1) / (each * per));
    if (cost < best) {
      best = cost;
      slices = (blocks + each * per - 1) / (each * per);
    }
    if (z == most) break;
  }
  const int each = (blocks + slices - 1) / slices;
  slices = (blocks + each - 1) / each;
  return {slices, slices * per, each * 128};
}

// Whether the pages' kernels read the prefix themselves, once per beam: while
// that is little they need no second kernel, no workspace and no join (32/8
// heads of 128: 16 beams over 128 keys 11.3 -> 6.4 us, 64 over 64 12.6 -> 7.6,
// even at 64 over 256; 16 over 512 13.9 against 12.4 us, 64 over 512 28 against
// 16; fp32, 8/8 heads of 64: 4 over 64 14.4 -> 6.8, 64 over 128 17.5 -> 13.7, 64
// over 256 20 against 18, 256 over 128 35 against 24).
constexpr int64_t PG_INLINE_BYTES = 64 << 20;   // of K and V, over all beams
constexpr int PG_INLINE_KEYS = 256;
static bool prefix_inline(int batch, int kv_heads, int D, int num_prefix, int item) {
  return num_prefix <= PG_INLINE_KEYS &&
         (int64_t)batch * num_prefix * kv_heads * D * 2 * item < PG_INLINE_BYTES;
}

// Slices of each beam's pages: enough CTAs of a long table to fill 148 SMs
// four times when there are few beams, none for less than 256 tokens (by the
// table's width: the lengths are on the device, and slices past a beam's length
// have no keys).  They are joined by a kernel of its own when they are cut, or when there are so many
// CTAs that those which wait for the prefix kernel to join it would keep the
// rest from the SMs it leaves free (512 beams x 8 K/V heads over 16384 keys: 179
// -> 168 us; 200 x 8 over 2048 keys: 39 against 41 us, so not there).
constexpr int PG_BESIDE = 2048;
struct PagesPlan {
  int slices;
  bool separate;
};
static PagesPlan pages_plan(int batch, int heads, int kv_heads, int num_prefix, int64_t room) {
  const int group = heads / kv_heads;
  const int64_t tasks = (int64_t)batch * kv_heads * ((group + PG_HEADS - 1) / PG_HEADS);
  const int64_t want = (4 * 148 + tasks - 1) / tasks;
  const int slices =
      (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, 64), room / 256));
  return {slices, slices > 1 || (num_prefix > 0 && room > 0 && tasks > PG_BESIDE)};
}

static bool aligned(const void* p, int64_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// 16-byte pieces of query, cache and current rows, 8-byte pieces of the output
static bool pages_mma_takes(const PagesArgs<__nv_bfloat16>& p) {
  if (p.prefix > 0 && !(aligned(p.pk, 16) && aligned(p.pv, 16) && p.pk_st % 8 == 0 &&
                        p.pk_sh % 8 == 0 && p.pv_st % 8 == 0 && p.pv_sh % 8 == 0))
    return false;
  return p.D % 8 == 0 && p.D <= 128 && aligned(p.q, 16) && p.q_sb % 8 == 0 && p.q_sh % 8 == 0 &&
         aligned(p.kc, 16) && aligned(p.vc, 16) && p.kc_sp % 8 == 0 && p.kc_st % 8 == 0 &&
         p.kc_sh % 8 == 0 && aligned(p.ck, 16) && aligned(p.cv, 16) && p.ck_sb % 8 == 0 &&
         p.ck_sh % 8 == 0 && aligned(p.out, 8) && p.o_sb % 4 == 0 && p.o_sh % 4 == 0;
}

template <int DP, bool kFew>
static int pages_mma_run(const PagesArgs<__nv_bfloat16>& p, int page_slices, bool after_prefix,
                         cudaStream_t stream) {
  const int64_t tasks = (int64_t)p.batch * p.kv_heads * ((p.group + PG_HEADS - 1) / PG_HEADS);
  if (tasks > INT_MAX || page_slices > 65535) return GRS_ERR_SHAPE;
  // warps of a CTA: a run of 32 tokens each, more when there are few CTAs
  const int64_t runs = ((int64_t)p.prefix + (int64_t)p.max_blocks * p.page + 1 + 31) / 32;
  const int warps = runs <= 2 && tasks * page_slices >= 4 * 148 ? 2 : tasks * page_slices >= 2 * 148 ? 4 : 8;
  constexpr int kRow = ((kFew ? 8 : PG_HEADS) * (PgShape<DP>::kStride + 2) + 32 * 4 + 2) * 4;
  const int smem = warps * kRow;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(pages_mma_kernel<DP, kFew>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           8 * kRow) != cudaSuccess)
    return GRS_ERR_CUDA;
  // starts under the prefix kernel's tail; its join waits for the slices
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)tasks, page_slices);
  config.blockDim = dim3(32 * warps);
  config.dynamicSmemBytes = smem;
  config.stream = counted(stream);
  config.attrs = &attr;
  config.numAttrs = after_prefix ? 1 : 0;
  if (cudaLaunchKernelEx(&config, pages_mma_kernel<DP, kFew>, p) != cudaSuccess)
    return GRS_ERR_CUDA;
  if (p.page_part) {
    const int parts = p.slices + page_slices, team = parts > 8 ? 4 : 1;
    const int64_t n = (int64_t)p.batch * p.heads;
    if (n > INT_MAX) return GRS_ERR_SHAPE;
    config.gridDim = dim3((unsigned)((n + 4 / team - 1) / (4 / team)));
    config.blockDim = dim3(128);
    config.dynamicSmemBytes = 0;
    config.stream = counted(stream);
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, join_parts_kernel, p, parts, team) != cudaSuccess)
      return GRS_ERR_CUDA;
  }
  GRS_CUDA_CHECK_LAUNCH();
  return GRS_OK;
}

static int pages_mma_launch(const PagesArgs<__nv_bfloat16>& p, int page_slices, bool after_prefix,
                            cudaStream_t stream) {
  const auto run = [&](auto few) {
    constexpr bool kFew = decltype(few)::value;
    if (p.D <= 32) return pages_mma_run<32, kFew>(p, page_slices, after_prefix, stream);
    if (p.D <= 64) return pages_mma_run<64, kFew>(p, page_slices, after_prefix, stream);
    return pages_mma_run<128, kFew>(p, page_slices, after_prefix, stream);
  };
  return p.group <= 8 ? run(std::true_type{}) : run(std::false_type{});
}

template <typename T>
static int shared_prefix(const PagesArgs<T>& p, const GroupedArgs<T>& prefix, bool tensor_cores,
                         int page_slices, cudaStream_t stream) {
  if (prefix.slices > 0) {
    int status = GRS_OK;
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      status = tensor_cores ? grouped_tc_launch(prefix, stream)
                            : grouped_rows_launch<T>(prefix, stream);
    else
      status = grouped_rows_launch<T>(prefix, stream);
    if (status != GRS_OK) return status;
  }
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    if (pages_mma_takes(p)) return pages_mma_launch(p, page_slices, prefix.slices > 0, stream);
  return pages_rows_launch<T>(p, prefix.slices > 0, stream);
}

}  // namespace grs

extern "C" int64_t grs_shared_prefix_workspace_bytes(int batch, int heads, int kv_heads,
                                                     int head_width, int num_prefix,
                                                     int64_t page_tokens) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 0;
  // any of the kernels may take the call, by the type and alignment of its tensors
  const auto parts = [&](int sliced, int64_t room) {
    const grs::PagesPlan pages = grs::pages_plan(batch, heads, kv_heads, sliced, room);
    return std::max(grs::rows_plan(batch, heads / kv_heads, kv_heads, head_width, sliced).parts,
                    grs::tc_plan(batch, heads, kv_heads, head_width, sliced).parts) +
           (pages.separate ? pages.slices : 0);
  };
  int most = 0;
  if (grs::prefix_inline(batch, kv_heads, head_width, num_prefix, 2))
    most = parts(0, page_tokens + num_prefix);
  if (!grs::prefix_inline(batch, kv_heads, head_width, num_prefix, 4))
    most = std::max(most, parts(num_prefix, page_tokens));
  return (int64_t)most * batch * heads * (head_width + 1) * 4;
}

extern "C" int grs_shared_prefix_attention(
    int dtype, const void* query, int64_t q_sb, int64_t q_sh, const void* prefix_key, int64_t pk_st,
    int64_t pk_sh, const void* prefix_value, int64_t pv_st, int64_t pv_sh, int num_prefix,
    const void* key_cache, const void* value_cache, int64_t kc_sp, int64_t kc_st, int64_t kc_sh,
    const int32_t* block_table, int64_t bt_stride, int max_blocks, const int32_t* lengths,
    int num_pages, int page_size, const void* current_key, const void* current_value,
    int64_t ck_sb, int64_t ck_sh, const uint8_t* current_valid, void* output, int64_t o_sb,
    int64_t o_sh, int batch, int heads, int kv_heads, int head_width, float scale, void* workspace,
    int64_t workspace_bytes, int32_t* status, void* stream) {
  using namespace grs;
  constexpr int kMost = 1 << 30;             // a tile's rows and a slice's keys add two places
  if (batch < 0 || batch >= kMost || heads <= 0 || heads >= kMost || kv_heads <= 0 ||
      heads % kv_heads || head_width <= 0 || head_width > 256 || !std::isfinite(scale * GA_LOG2E) ||
      num_prefix < 0 || num_prefix >= kMost || max_blocks < 0 || num_pages < 0 ||
      (max_blocks > 0 && (page_size <= 0 || !block_table || !lengths ||
                          (int64_t)max_blocks * page_size > INT_MAX / 2)) ||
      (max_blocks > 0 && num_pages > 0 && (!key_cache || !value_cache)) ||
      (num_prefix > 0 && (!prefix_key || !prefix_value)) || (current_key && !current_value))
    return GRS_ERR_SHAPE;
  if (batch == 0) return GRS_OK;
  if (!query || !output) return GRS_ERR_SHAPE;
  const int64_t room = (int64_t)max_blocks * page_size;
  const int64_t need = grs_shared_prefix_workspace_bytes(batch, heads, kv_heads, head_width,
                                                         num_prefix, room);
  if (need > 0 && (!workspace || workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return GRS_ERR_WORKSPACE;
  const int group = heads / kv_heads;
  const float scale_log2 = scale * GA_LOG2E;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    GroupedArgs<T> g = {};
    g.q = static_cast<const T*>(query); g.q_sp = q_sb; g.q_sh = q_sh;
    g.k = static_cast<const T*>(prefix_key); g.k_st = pk_st; g.k_sh = pk_sh;
    g.v = static_cast<const T*>(prefix_value); g.v_st = pv_st; g.v_sh = pv_sh;
    g.positions = batch; g.keys = num_prefix; g.heads = heads; g.kv_heads = kv_heads;
    g.group = group; g.D = head_width; g.scale_log2 = scale_log2;
    const bool inlined =
        prefix_inline(batch, kv_heads, head_width, num_prefix, (int)sizeof(T));
    const int sliced = inlined ? 0 : num_prefix;
    bool tensor_cores = false;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) tensor_cores = grouped_tc_takes(g);
    const PrefixPlan plan = tensor_cores ? tc_plan(batch, heads, kv_heads, head_width, sliced)
                                         : rows_plan(batch, group, kv_heads, head_width, sliced);
    float* part = static_cast<float*>(workspace);
    const PagesPlan pages =
        pages_plan(batch, heads, kv_heads, sliced, room + (inlined ? num_prefix : 0));
    const int64_t parts = plan.parts + (pages.separate ? pages.slices : 0);
    float* lse = part + parts * batch * heads * head_width;
    g.part = part; g.part_lse = lse; g.slices = plan.slices; g.slice_keys = plan.keys;
    g.status = status;
    PagesArgs<T> p = {};
    p.q = g.q; p.q_sb = q_sb; p.q_sh = q_sh;
    p.kc = static_cast<const T*>(key_cache); p.vc = static_cast<const T*>(value_cache);
    p.kc_sp = kc_sp; p.kc_st = kc_st; p.kc_sh = kc_sh;
    p.bt = block_table; p.bt_s = bt_stride; p.max_blocks = max_blocks;
    p.lengths = lengths; p.num_pages = num_pages; p.page = page_size;
    p.ck = static_cast<const T*>(current_key); p.cv = static_cast<const T*>(current_value);
    p.ck_sb = ck_sb; p.ck_sh = ck_sh; p.cvalid = current_valid;
    if (inlined) {
      p.pk = g.k; p.pk_st = pk_st; p.pk_sh = pk_sh;
      p.pv = g.v; p.pv_st = pv_st; p.pv_sh = pv_sh;
      p.prefix = num_prefix;
    }
    p.part = part; p.part_lse = lse;
    p.slices = plan.parts;
    if (pages.separate) {
      p.page_part = part;
      p.page_lse = lse;
    }
    p.out = static_cast<T*>(output); p.o_sb = o_sb; p.o_sh = o_sh;
    p.batch = batch; p.heads = heads; p.kv_heads = kv_heads; p.group = group; p.D = head_width;
    p.scale_log2 = scale_log2; p.status = status;
    return shared_prefix<T>(p, g, tensor_cores, pages.slices, s);
  };
  if (dtype == GRS_DTYPE_F32) return go(float{});
  if (dtype == GRS_DTYPE_BF16) return go(__nv_bfloat16{});
  return GRS_ERR_SHAPE;
}
