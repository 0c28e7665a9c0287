// Penalties for repeated tokens, biases and grammar masks on next-token
// logits: grs_adjust_logits.
//
// One pass, bound by HBM.  A CTA takes a run of one row's vocabulary in blocks
// of two 16-byte vectors a thread, requesting the next block's logits, mask
// words and biases before it writes the present one (a vector whose mask bits
// are all clear is written without being read).  Under the first block's loads
// it counts the row's history tokens that fall into the run in shared memory:
// whole numbers, so the order of the atomics does not matter.  Every run reads
// the whole history, so runs are long where that leaves enough CTAs.
// Blocks start on 16-byte boundaries of the row's address, so rows of any
// alignment take full vectors but for their first and last.  256 x 150000 fp32
// logits with a bias per row and histories of 4096 take 82 us, 5.65 TB/s or 0.87
// of the measured copy; 1000 x 32003 bf16 logits with a mask 32 us, 4.0 TB/s.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "grs_common.cuh"

namespace grs {

struct LogitsArgs {
  const void* logits; int64_t l_sb;
  void* out; int64_t o_sb;
  int rows, vocab;
  const void* tokens; int64_t t_sb; int history;
  const int32_t* lengths; const int32_t* prompt_lengths;
  const float* repetition; const float* presence; const float* frequency;   // [rows] or null
  float repetition_all, presence_all, frequency_all;
  const float* bias; int64_t b_sb;
  const int32_t* allowed; int64_t a_sb;
  float fill;
};

constexpr int TL_THREADS = 256;

template <typename T>
__device__ __forceinline__ uint4 tl_pack(const float* x) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                      __float_as_uint(x[3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Counts per column: bit 0: seen anywhere in the history; the rest: times
// generated.  Two columns share a word while the history is below 2^14, so that
// 2 * count + 1 fits 16 bits.
constexpr int TL_NARROW = 1 << 14;

// Blocks of a run.  Longer runs read the history fewer times, their counters
// leave room for fewer CTAs: 1 / 2 / 4 / 8 blocks took 122 / 93 / 82 / 80 us on
// 256 x 150000 fp32 with histories of 4096 and 41 / 33 / 31 / 38 us on 1000 x
// 32003 bf16 with histories of 64.
constexpr int TL_LONGEST = 4;

template <bool kNarrow>
__device__ __forceinline__ void tl_count(uint32_t* seen, int at, bool generated) {
  const int move = kNarrow ? 16 * (at & 1) : 0;
  uint32_t* word = seen + (kNarrow ? at >> 1 : at);
  if (generated) atomicAdd(word, 2u << move); else atomicOr(word, 1u << move);
}

template <typename T, bool kBias>
struct TlBlock {
  static constexpr int W = 16 / sizeof(T);
  uint4 x[2];
  float bias[kBias ? 2 : 1][kBias ? W : 1];
  uint32_t open[2];    // allowed columns of the vector; from bit 16 on: columns in the row
};

// Block k of a run covers the columns lo + (2 k + i) * threads * W + tid * W ...
// for i = 0, 1, where lo is the run's first column less the row's first
// element's place in its 16 bytes.
template <typename T, typename Tok, bool kNarrow, bool kBias>
__global__ void __launch_bounds__(TL_THREADS, kBias ? 3 : 4)
adjust_logits_kernel(LogitsArgs a, int runs, int blocks) {
  using B = TlBlock<T, kBias>;
  constexpr int W = B::W, kVector = TL_THREADS * W;
  constexpr uint32_t kAll = (1u << W) - 1u;
  extern __shared__ __align__(16) uint32_t seen[];
  const int row = blockIdx.x / runs, tid = threadIdx.x;
  const T* in = static_cast<const T*>(a.logits) + row * a.l_sb;
  T* out = static_cast<T*>(a.out) + row * a.o_sb;
  const int shift = (int)(reinterpret_cast<uintptr_t>(in) & 15) / (int)sizeof(T);
  const bool same = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const int span = blocks * 2 * kVector;
  const int lo = (blockIdx.x % runs) * span - shift;
  const int32_t* allowed = a.allowed ? a.allowed + row * a.a_sb : nullptr;
  const float* bias = kBias ? a.bias + row * a.b_sb : nullptr;
  int len = 0, prompt = 0;
  if (a.tokens) {
    len = a.lengths ? min(max(a.lengths[row], 0), a.history) : a.history;
    prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
  }
  const float rep = a.repetition ? a.repetition[row] : a.repetition_all;
  const float pres = a.presence ? a.presence[row] : a.presence_all;
  const float freq = a.frequency ? a.frequency[row] : a.frequency_all;

  const auto fetch = [&](B& f, int block) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int v = lo + (2 * block + i) * kVector + tid * W;
      uint32_t in_row = kAll;
      if (v < 0) in_row &= kAll & ~((1u << -v) - 1u);        // -v = shift < W
      if (v > a.vocab - W) in_row &= a.vocab > v ? (1u << (a.vocab - v)) - 1u : 0u;
      uint32_t open = in_row;
      if (allowed && in_row) {
        const int first = max(v, 0), last = min(v + W, a.vocab) - 1;
        const uint32_t w0 = (uint32_t)__ldg(allowed + (first >> 5));
        const uint32_t w1 = (uint32_t)__ldg(allowed + (last >> 5));
        open &= __funnelshift_r(w0, w1, first & 31) << (first - v);
      }
      f.open[i] = open | in_row << 16;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int v = lo + (2 * block + i) * kVector + tid * W;
      const uint32_t in_row = f.open[i] >> 16;
      f.x[i] = make_uint4(0, 0, 0, 0);
      if ((f.open[i] & kAll) == 0) continue;
      if (in_row == kAll) {
        f.x[i] = __ldcs(reinterpret_cast<const uint4*>(in + v));
      } else {
        float y[W];
#pragma unroll
        for (int j = 0; j < W; ++j) y[j] = (in_row >> j) & 1 ? to_float(in[v + j]) : 0.f;
        f.x[i] = tl_pack<T>(y);
      }
      if constexpr (kBias) {
        if (in_row == kAll && (reinterpret_cast<uintptr_t>(bias + v) & 15) == 0) {
#pragma unroll
          for (int j = 0; j < W; j += 4) {
            const float4 b = __ldg(reinterpret_cast<const float4*>(bias + v + j));
            f.bias[i][j] = b.x;
            f.bias[i][j + 1] = b.y;
            f.bias[i][j + 2] = b.z;
            f.bias[i][j + 3] = b.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j)
            f.bias[i][j] = (in_row >> j) & 1 ? __ldg(bias + v + j) : 0.f;
        }
      }
    }
  };

  B now;
  fetch(now, 0);
  if (len > 0) {
    const int vectors = span / (kNarrow ? 8 : 4);
    for (int i = tid; i < vectors; i += TL_THREADS)
      reinterpret_cast<uint4*>(seen)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const Tok* tokens = static_cast<const Tok*>(a.tokens) + row * a.t_sb;
    // (a negative id may reach the places before the row's first column, which
    // nothing looks up; the difference is exact or far out of the run)
    using U = std::make_unsigned_t<Tok>;
    for (int i0 = tid; i0 < len; i0 += 8 * TL_THREADS) {
      U at[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = i0 + j * TL_THREADS;
        at[j] = i < len ? (U)__ldg(tokens + i) - (U)(Tok)lo : ~(U)0;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at[j] < (U)span) tl_count<kNarrow>(seen, (int)at[j], i0 + j * TL_THREADS >= prompt);
    }
    __syncthreads();
  }

  for (int block = 0; block < blocks; ++block) {
    B next;
    if (block + 1 < blocks) fetch(next, block + 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = (2 * block + i) * kVector + tid * W, v = lo + at;
      const uint32_t in_row = now.open[i] >> 16;
      if (!in_row) continue;
      const uint32_t* words = reinterpret_cast<const uint32_t*>(&now.x[i]);
      float y[W];
#pragma unroll
      for (int j = 0; j < W; ++j)
        y[j] = sizeof(T) == 4 ? __uint_as_float(words[j])
                              : __uint_as_float(j & 1 ? words[j / 2] & 0xffff0000u
                                                      : words[j / 2] << 16);
      if (len > 0) {
        uint32_t counts[kNarrow ? W / 2 : W];
        uint32_t any = 0;
#pragma unroll
        for (int j = 0; j < (kNarrow ? W / 2 : W); ++j) {
          counts[j] = seen[(kNarrow ? at >> 1 : at) + j];
          any |= counts[j];
        }
        if (any) {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const uint32_t c = kNarrow ? (counts[j / 2] >> (16 * (j & 1))) & 0xffffu : counts[j];
            if (c) {
              y[j] = y[j] > 0.f ? y[j] / rep : y[j] * rep;
              if (c > 1) y[j] = y[j] - freq * (float)(c >> 1) - pres;
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < W; ++j) {
        if constexpr (kBias) y[j] += now.bias[i][j];
        if (!((now.open[i] >> j) & 1)) y[j] = a.fill;
      }
      if (in_row == kAll && same) {
        __stcs(reinterpret_cast<uint4*>(out + v), tl_pack<T>(y));
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
          if ((in_row >> j) & 1) out[v + j] = from_float<T>(y[j]);
      }
    }
    now = next;
  }
}

template <typename T, typename Tok, bool kNarrow, bool kBias>
static int adjust_logits_launch(const LogitsArgs& a, cudaStream_t stream) {
  constexpr int W = 16 / sizeof(T), kBlock = 2 * TL_THREADS * W;
  const int all = (a.vocab + W - 1 + kBlock - 1) / kBlock;    // blocks of a row, any shift
  // shorter runs where the longest would give fewer than four CTAs per SM
  const int64_t most = std::max<int64_t>(1, (int64_t)all * a.rows / (4 * 148));
  int blocks = (int)std::min<int64_t>(TL_LONGEST, most);
  int runs = (all + blocks - 1) / blocks;
  blocks = (all + runs - 1) / runs;
  if ((int64_t)runs * a.rows > INT_MAX) return GRS_ERR_SHAPE;
  const int smem = a.tokens ? blocks * kBlock * (kNarrow ? 2 : 4) : 0;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(adjust_logits_kernel<T, Tok, kNarrow, kBias>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return GRS_ERR_CUDA;
  adjust_logits_kernel<T, Tok, kNarrow, kBias>
      <<<(unsigned)(runs * a.rows), TL_THREADS, smem, counted(stream)>>>(a, runs, blocks);
  GRS_CUDA_CHECK_LAUNCH();
  return GRS_OK;
}

template <typename T, typename Tok>
static int adjust_logits_counts(const LogitsArgs& a, cudaStream_t stream) {
  if (a.history < TL_NARROW)
    return a.bias ? adjust_logits_launch<T, Tok, true, true>(a, stream)
                  : adjust_logits_launch<T, Tok, true, false>(a, stream);
  return a.bias ? adjust_logits_launch<T, Tok, false, true>(a, stream)
                : adjust_logits_launch<T, Tok, false, false>(a, stream);
}

}  // namespace grs

extern "C" int grs_adjust_logits(int dtype, const void* logits, int64_t l_sb, void* out,
                                 int64_t o_sb, int rows, int vocab, const void* tokens,
                                 int tokens_are_i64, int64_t t_sb, int history,
                                 const int32_t* lengths, const int32_t* prompt_lengths,
                                 const float* repetition, const float* presence,
                                 const float* frequency, float repetition_all, float presence_all,
                                 float frequency_all, const float* bias, int64_t bias_sb,
                                 const int32_t* allowed, int64_t a_sb, float fill, void* stream) {
  using namespace grs;
  if (rows < 0 || vocab < 0 || history < 0 || history >= (1 << 30) || vocab >= (1 << 30) ||
      (dtype != GRS_DTYPE_BF16 && dtype != GRS_DTYPE_F32))
    return GRS_ERR_SHAPE;
  if (rows == 0 || vocab == 0) return GRS_OK;
  if (!logits || !out || (history > 0 && !tokens)) return GRS_ERR_SHAPE;
  LogitsArgs a;
  a.logits = logits; a.l_sb = l_sb; a.out = out; a.o_sb = o_sb; a.rows = rows; a.vocab = vocab;
  a.tokens = history > 0 ? tokens : nullptr; a.t_sb = t_sb; a.history = history;
  a.lengths = lengths; a.prompt_lengths = prompt_lengths;
  a.repetition = repetition; a.presence = presence; a.frequency = frequency;
  a.repetition_all = repetition_all; a.presence_all = presence_all;
  a.frequency_all = frequency_all;
  a.bias = bias; a.b_sb = bias_sb; a.allowed = allowed; a.a_sb = a_sb; a.fill = fill;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == GRS_DTYPE_BF16)
    return tokens_are_i64 ? adjust_logits_counts<__nv_bfloat16, int64_t>(a, s)
                          : adjust_logits_counts<__nv_bfloat16, int32_t>(a, s);
  return tokens_are_i64 ? adjust_logits_counts<float, int64_t>(a, s)
                        : adjust_logits_counts<float, int32_t>(a, s);
}
