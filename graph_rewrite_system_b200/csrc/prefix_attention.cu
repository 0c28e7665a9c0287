// One query per beam against a prefix that every beam shares and against the
// beam's own pages: grs_shared_prefix_attention.
//
// The prefix is attention of beams * group rows per K/V head to the same keys,
// so its K/V are read once per tile of rows instead of once per beam; it is cut
// into slices when the tiles alone would leave SMs idle.  Each slice leaves its
// normalised fp32 sum and log2 weight in the workspace; the pages kernel adds
// the beam's own keys, joins all parts by their weights and writes the output.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "grouped_attention_tc.cuh"

namespace grs {

template <typename T>
struct PagesArgs {
  const T* q; int64_t q_sb, q_sh;
  const T* kc; const T* vc; int64_t kc_sp, kc_st, kc_sh;
  const int32_t* bt; int64_t bt_s; int max_blocks; const int32_t* lengths; int num_pages, page;
  const T* ck; const T* cv; int64_t ck_sb, ck_sh; const uint8_t* cvalid;
  const float* part; const float* part_lse; int slices;
  T* out; int64_t o_sb, o_sh;
  int batch, heads, kv_heads, group, D;
  float scale_log2;
  int32_t* status;
};

// One warp per (beam, head): online softmax over 32-key steps, a lane per key
// for the scores and a lane per dimension for the values, then the join with
// the prefix slices.
template <typename T, int DP>
__global__ void __launch_bounds__(128) pages_rows_kernel(PagesArgs<T> a) {
  constexpr int ND = (DP + 31) / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (int64_t)a.batch * a.heads) return;
  const int b = (int)(row / a.heads), head = (int)(row % a.heads), h = head / a.group;
  const T* q = a.q + (int64_t)b * a.q_sb + (int64_t)head * a.q_sh;

  const int room = a.max_blocks * a.page;
  int past = a.lengths ? a.lengths[b] : 0;
  if (past < 0 || past > room) {
    if (lane == 0) set_status(a.status, GRS_ERR_LENGTH);
    past = min(max(past, 0), room);
  }
  const bool cur = a.ck != nullptr && (a.cvalid == nullptr || a.cvalid[b] != 0);
  const int total = past + (cur ? 1 : 0);
  // element offset of token t's row, or -1 when its page is not in the cache
  const auto place = [&](int t) -> int64_t {
    const int page = a.bt[(int64_t)b * a.bt_s + t / a.page];
    if (page < 0 || page >= a.num_pages) {
      set_status(a.status, GRS_ERR_BAD_PAGE);
      return -1;
    }
    return (int64_t)page * a.kc_sp + (int64_t)(t % a.page) * a.kc_st + (int64_t)h * a.kc_sh;
  };

  float m = -INFINITY, l = 0.f, acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = 0.f;
  for (int t0 = 0; t0 < total; t0 += 32) {
    const int t = t0 + lane;
    int64_t at = -1;
    const T* k = nullptr;
    if (t < past) {
      at = place(t);
      if (at >= 0) k = a.kc + at;
    } else if (t < total) {
      k = a.ck + (int64_t)b * a.ck_sb + (int64_t)h * a.ck_sh;
    }
    float s = -INFINITY;
    if (k) {
      float dot = 0.f;
      for (int d = 0; d < a.D; ++d) dot = fmaf(to_float(q[d]), to_float(k[d]), dot);
      s = dot * a.scale_log2;
    }
    const float top = fmaxf(m, warp_max(s));
    const float base = top == -INFINITY ? 0.f : top;
    const float w = exp2f(s - base);
    const float keep = exp2f(m - base);
    l = l * keep + warp_sum(w);
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] *= keep;
    m = top;
    const int n = min(32, total - t0);
    for (int j = 0; j < n; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const int64_t vat = __shfl_sync(0xffffffffu, at, j);
      const bool is_cur = t0 + j >= past;
      if (vat < 0 && !is_cur) continue;
      const T* v = is_cur ? a.cv + (int64_t)b * a.ck_sb + (int64_t)h * a.ck_sh : a.vc + vat;
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const int d = lane + 32 * i;
        if (d < a.D) acc[i] = fmaf(wj, to_float(v[d]), acc[i]);
      }
    }
  }

  // join: weights exp2(lse_i - max lse); the pages' sum enters unnormalised
  float top = m;
  for (int i = lane; i < a.slices; i += 32)
    top = fmaxf(top, a.part_lse[((int64_t)i * a.batch + b) * a.heads + head]);
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  const float own = exp2f(m - base);
  float norm = l * own;
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] *= own;
#pragma unroll 4
  for (int i = 0; i < a.slices; ++i) {
    const int64_t at = ((int64_t)i * a.batch + b) * a.heads + head;
    const float w = exp2f(a.part_lse[at] - base);
    norm += w;
#pragma unroll
    for (int j = 0; j < ND; ++j) {
      const int d = lane + 32 * j;
      if (d < a.D) acc[j] = fmaf(w, a.part[at * a.D + d], acc[j]);
    }
  }
  const float inv = norm == 0.f ? 0.f : 1.f / norm;
  T* o = a.out + (int64_t)b * a.o_sb + (int64_t)head * a.o_sh;
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int d = lane + 32 * i;
    if (d < a.D) o[d] = from_float<T>(acc[i] * inv);
  }
}

// How the prefix is cut: `parts` partial sums, `keys` per slice (two parts per
// slice when the tensor-core kernel's slots halve it).
struct PrefixPlan {
  int slices, parts, keys;
};

// fp32 rows: enough CTAs for two waves of 148 SMs, none shorter than 256 keys.
static PrefixPlan rows_plan(int batch, int group, int kv_heads, int keys) {
  if (keys <= 0) return {0, 0, 0};
  const int64_t tiles = ((int64_t)batch * group + 63) / 64 * kv_heads;
  const int64_t want =
      std::max<int64_t>(1, std::min<int64_t>((2 * 148 + tiles - 1) / tiles, (keys + 255) / 256));
  const int each = (int)(((keys + want - 1) / want + 127) / 128 * 128);
  const int slices = (keys + each - 1) / each;
  return {slices, slices, each};
}

// Tensor cores: the count whose waves of 148 CTAs take the fewest 128-key
// blocks, each wave paying about four blocks for its start and end and every
// part the write and read of its fp32 sums (a block takes about 1.1 us).
static PrefixPlan tc_plan(int batch, int heads, int kv_heads, int D, int keys) {
  if (keys <= 0) return {0, 0, 0};
  const int group = heads / kv_heads;
  const bool split = grouped_tc_split(batch, group);
  const int pps = std::max(1, 128 / group) * (split ? 1 : 2);
  const int64_t tiles = ((int64_t)batch + pps - 1) / pps * kv_heads;
  // slots of a split slice take turns on half the blocks each
  const int blocks = (keys + 127) / 128, per = split ? 2 : 1;
  const double join = 8.0 * batch * heads * D / 6.5e12 / 1.1e-6 + 0.02;
  double best = 1e30;
  int slices = 1;
  for (int z = 1; z <= std::min(64, (blocks + per - 1) / per); ++z) {
    const int64_t waves = (tiles * z + 147) / 148;
    const int64_t each = ((blocks + z - 1) / z + per - 1) / per;
    const double cost = (double)waves * (each + 4) + join * z * per;
    if (cost < best) {
      best = cost;
      slices = z;
    }
  }
  const int each = (blocks + slices - 1) / slices;
  slices = (blocks + each - 1) / each;
  return {slices, slices * per, each * 128};
}

static size_t plan_bytes(const PrefixPlan& p, int batch, int heads, int D) {
  return (size_t)p.parts * batch * heads * (D + 1) * 4;
}

template <typename T>
static int shared_prefix(const PagesArgs<T>& p, const GroupedArgs<T>& prefix, bool tensor_cores,
                         cudaStream_t stream) {
  if (prefix.slices > 0) {
    int status = GRS_OK;
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      status = tensor_cores ? grouped_tc_launch(prefix, stream)
                            : grouped_rows_launch<T>(prefix, stream);
    else
      status = grouped_rows_launch<T>(prefix, stream);
    if (status != GRS_OK) return status;
  }
  const int64_t rows = (int64_t)p.batch * p.heads;
  const unsigned grid = (unsigned)((rows + 3) / 4);
  if (p.D <= 32) pages_rows_kernel<T, 32><<<grid, 128, 0, counted(stream)>>>(p);
  else if (p.D <= 64) pages_rows_kernel<T, 64><<<grid, 128, 0, counted(stream)>>>(p);
  else if (p.D <= 128) pages_rows_kernel<T, 128><<<grid, 128, 0, counted(stream)>>>(p);
  else pages_rows_kernel<T, 256><<<grid, 128, 0, counted(stream)>>>(p);
  GRS_CUDA_CHECK_LAUNCH();
  return GRS_OK;
}

}  // namespace grs

extern "C" int64_t grs_shared_prefix_workspace_bytes(int batch, int heads, int kv_heads,
                                                     int head_width, int num_prefix) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || num_prefix <= 0) return 0;
  // either kernel may take the call, by the alignment of its tensors
  return (int64_t)std::max(
      grs::plan_bytes(grs::rows_plan(batch, heads / kv_heads, kv_heads, num_prefix), batch, heads,
                      head_width),
      grs::plan_bytes(grs::tc_plan(batch, heads, kv_heads, head_width, num_prefix), batch, heads,
                      head_width));
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
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_width <= 0 ||
      head_width > 256 || !std::isfinite(scale) || num_prefix < 0 || max_blocks < 0 || num_pages < 0 ||
      (max_blocks > 0 && (page_size <= 0 || !block_table || !lengths || !key_cache ||
                          !value_cache || (int64_t)max_blocks * page_size > INT_MAX / 2)) ||
      (num_prefix > 0 && (!prefix_key || !prefix_value)) || (current_key && !current_value))
    return GRS_ERR_SHAPE;
  if (batch == 0) return GRS_OK;
  if (!query || !output) return GRS_ERR_SHAPE;
  const int64_t need =
      grs_shared_prefix_workspace_bytes(batch, heads, kv_heads, head_width, num_prefix);
  if (need > 0 && (!workspace || workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return GRS_ERR_WORKSPACE;
  const int group = heads / kv_heads;
  const float scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    GroupedArgs<T> g = {};
    g.q = static_cast<const T*>(query); g.q_sp = q_sb; g.q_sh = q_sh;
    g.k = static_cast<const T*>(prefix_key); g.k_st = pk_st; g.k_sh = pk_sh;
    g.v = static_cast<const T*>(prefix_value); g.v_st = pv_st; g.v_sh = pv_sh;
    g.positions = batch; g.keys = num_prefix; g.heads = heads; g.kv_heads = kv_heads;
    g.group = group; g.D = head_width; g.scale_log2 = scale_log2;
    bool tensor_cores = false;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) tensor_cores = grouped_tc_takes(g);
    const PrefixPlan plan = tensor_cores ? tc_plan(batch, heads, kv_heads, head_width, num_prefix)
                                         : rows_plan(batch, group, kv_heads, num_prefix);
    float* part = static_cast<float*>(workspace);
    float* lse = plan.parts ? part + (size_t)plan.parts * batch * heads * head_width : nullptr;
    g.part = part; g.part_lse = lse; g.slices = plan.slices; g.slice_keys = plan.keys;
    g.status = status;
    PagesArgs<T> p = {};
    p.q = g.q; p.q_sb = q_sb; p.q_sh = q_sh;
    p.kc = static_cast<const T*>(key_cache); p.vc = static_cast<const T*>(value_cache);
    p.kc_sp = kc_sp; p.kc_st = kc_st; p.kc_sh = kc_sh;
    p.bt = block_table; p.bt_s = bt_stride; p.max_blocks = max_blocks;
    p.lengths = max_blocks ? lengths : nullptr; p.num_pages = num_pages; p.page = page_size;
    p.ck = static_cast<const T*>(current_key); p.cv = static_cast<const T*>(current_value);
    p.ck_sb = ck_sb; p.ck_sh = ck_sh; p.cvalid = current_valid;
    p.part = part; p.part_lse = lse; p.slices = plan.parts;
    p.out = static_cast<T*>(output); p.o_sb = o_sb; p.o_sh = o_sh;
    p.batch = batch; p.heads = heads; p.kv_heads = kv_heads; p.group = group; p.D = head_width;
    p.scale_log2 = scale_log2; p.status = status;
    return shared_prefix<T>(p, g, tensor_cores, s);
  };
  if (dtype == GRS_DTYPE_F32) return go(float{});
  if (dtype == GRS_DTYPE_BF16) return go(__nv_bfloat16{});
  return GRS_ERR_SHAPE;
}
