// Causal attention over packed prompts: the host side of grs_prompt_attention.
#include <cmath>
#include <type_traits>

#include "grouped_attention_tc.cuh"

namespace grs {
namespace {

template <typename T>
int prompt_attention(const void* query, int64_t q_st, int64_t q_sh, const void* key, int64_t k_st,
                     int64_t k_sh, const void* value, int64_t v_st, int64_t v_sh,
                     const int32_t* offsets, int sequences, void* out, int64_t o_st, int64_t o_sh,
                     int tokens, int heads, int kv_heads, int head_width, float scale,
                     int clear_rest, int32_t* status, cudaStream_t stream) {
  GroupedArgs<T> a = {};
  a.q = static_cast<const T*>(query); a.q_sp = q_st; a.q_sh = q_sh;
  a.k = static_cast<const T*>(key); a.k_st = k_st; a.k_sh = k_sh;
  a.v = static_cast<const T*>(value); a.v_st = v_st; a.v_sh = v_sh;
  a.positions = a.keys = tokens;
  a.heads = heads; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.D = head_width;
  a.scale_log2 = scale * GA_LOG2E;
  a.offsets = offsets; a.sequences = sequences;
  a.out = static_cast<T*>(out); a.o_sp = o_st; a.o_sh = o_sh;
  a.clear_rest = clear_rest;
  a.status = status;
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    if (grouped_tc_takes(a)) return grouped_tc_launch(a, stream);
  return grouped_rows_launch<T>(a, stream);
}

}  // namespace
}  // namespace grs

extern "C" int grs_prompt_attention(int dtype, const void* query, int64_t q_st, int64_t q_sh,
                                    const void* key, int64_t k_st, int64_t k_sh,
                                    const void* value, int64_t v_st, int64_t v_sh,
                                    const int32_t* offsets, int sequences, void* out,
                                    int64_t o_st, int64_t o_sh, int tokens, int heads,
                                    int kv_heads, int head_width, float scale, int clear_rest,
                                    int32_t* status, void* stream) {
  // below 2^30: the search among the offsets and a tile's positions add two places
  constexpr int kMost = 1 << 30;
  if (tokens < 0 || tokens >= kMost || sequences < 0 || sequences >= kMost || heads <= 0 ||
      heads >= kMost || kv_heads <= 0 || heads % kv_heads || head_width <= 0 || head_width > 256 ||
      !std::isfinite(scale * grs::GA_LOG2E))
    return GRS_ERR_SHAPE;
  if (tokens == 0) return GRS_OK;
  if (!query || !key || !value || !offsets || !out) return GRS_ERR_SHAPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == GRS_DTYPE_F32)
    return grs::prompt_attention<float>(query, q_st, q_sh, key, k_st, k_sh, value, v_st, v_sh,
                                        offsets, sequences, out, o_st, o_sh, tokens, heads,
                                        kv_heads, head_width, scale, clear_rest, status, s);
  if (dtype == GRS_DTYPE_BF16)
    return grs::prompt_attention<__nv_bfloat16>(query, q_st, q_sh, key, k_st, k_sh, value, v_st,
                                                v_sh, offsets, sequences, out, o_st, o_sh, tokens,
                                                heads, kv_heads, head_width, scale, clear_rest,
                                                status, s);
  return GRS_ERR_SHAPE;
}
