// Penalties for repeated tokens, biases and grammar masks on next-token
// logits: grs_adjust_logits.
//
// One pass: a CTA takes a run of one row's vocabulary, counts the row's
// history tokens that fall into it in shared memory (whole numbers, so the
// order of the atomics does not matter), and writes the run's logits.  A
// masked logit is written without being read.
#include <climits>

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

constexpr int TL_RUN = 4096, TL_THREADS = 256;

template <typename T, typename Tok>
__global__ void __launch_bounds__(TL_THREADS) adjust_logits_kernel(LogitsArgs a) {
  // bit 0: seen anywhere in the history; the rest: times generated
  __shared__ int seen[TL_RUN];
  const int runs = (a.vocab + TL_RUN - 1) / TL_RUN;
  const int row = blockIdx.x / runs, tid = threadIdx.x;
  const int lo = (blockIdx.x % runs) * TL_RUN, n = min(TL_RUN, a.vocab - lo);
  int len = 0;
  if (a.tokens) {
    len = a.lengths ? min(max(a.lengths[row], 0), a.history) : a.history;
    const int prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    for (int i = tid; i < n; i += TL_THREADS) seen[i] = 0;
    __syncthreads();
    const Tok* tokens = static_cast<const Tok*>(a.tokens) + row * a.t_sb;
    for (int i = tid; i < len; i += TL_THREADS) {
      const int64_t at = (int64_t)tokens[i] - lo;
      if (at >= 0 && at < n) {
        if (i < prompt) atomicOr(&seen[at], 1); else atomicAdd(&seen[at], 2);
      }
    }
    __syncthreads();
  }
  const float rep = a.repetition ? a.repetition[row] : a.repetition_all;
  const float pres = a.presence ? a.presence[row] : a.presence_all;
  const float freq = a.frequency ? a.frequency[row] : a.frequency_all;
  const T* in = static_cast<const T*>(a.logits) + row * a.l_sb + lo;
  T* out = static_cast<T*>(a.out) + row * a.o_sb + lo;
  for (int i = tid; i < n; i += TL_THREADS) {
    const int v = lo + i;
    float x = a.fill;
    if (!a.allowed || ((a.allowed[row * a.a_sb + (v >> 5)] >> (v & 31)) & 1)) {
      x = to_float(in[i]);
      const int s = len ? seen[i] : 0;
      if (s) {
        x = x > 0.f ? x / rep : x * rep;
        const int count = s >> 1;
        if (count) x = x - freq * (float)count - pres;
      }
      if (a.bias) x += a.bias[row * a.b_sb + v];
    }
    out[i] = from_float<T>(x);
  }
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
  const int64_t ctas = (int64_t)((vocab + TL_RUN - 1) / TL_RUN) * rows;
  if (ctas > INT_MAX) return GRS_ERR_SHAPE;
  const unsigned grid = (unsigned)ctas;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == GRS_DTYPE_BF16) {
    if (tokens_are_i64)
      adjust_logits_kernel<__nv_bfloat16, int64_t><<<grid, TL_THREADS, 0, counted(s)>>>(a);
    else
      adjust_logits_kernel<__nv_bfloat16, int32_t><<<grid, TL_THREADS, 0, counted(s)>>>(a);
  } else {
    if (tokens_are_i64)
      adjust_logits_kernel<float, int64_t><<<grid, TL_THREADS, 0, counted(s)>>>(a);
    else
      adjust_logits_kernel<float, int32_t><<<grid, TL_THREADS, 0, counted(s)>>>(a);
  }
  GRS_CUDA_CHECK_LAUNCH();
  return GRS_OK;
}
