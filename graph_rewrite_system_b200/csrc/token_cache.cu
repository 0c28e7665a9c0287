// New keys and values into the pages of a paged cache, the keys (and the step's
// queries) turned by their positions on the way: grs_append_tokens.
#include <algorithm>
#include <climits>
#include <cmath>

#include "e4m3.cuh"
#include "rotary.cuh"

namespace grs {

struct AppendArgs {
  const void* q; int64_t q_st, q_sh; void* qo; int64_t qo_st, qo_sh;   // q may be null
  const void* k; int64_t k_st, k_sh;
  const void* v; int64_t v_st, v_sh;
  void* kc; void* vc; int64_t c_sp, c_st, c_sh;       // strides in elements
  float* ks; float* vs; int64_t s_sp;                 // scales [pages, kv_heads], or null
  const int32_t* table; int64_t t_s; const int32_t* source; int64_t source_s; int columns;
  const int32_t* lengths; const int32_t* offsets;     // offsets null: a token per sequence
  const void* positions; int wide;                    // int32 or int64 [tokens], or null
  const double* freq; int pairs; float magnitude, key_most;
  int tokens, sequences, group, kv_heads, width, pages, page;
  int units, heads_each, rows, clear;
  int32_t* status;
};

constexpr int AP_THREADS = 256;
constexpr int AP_ROWS = 16;                 // rows of a CTA's table of turns
constexpr int AP_AHEAD = 4;                 // units of a thread in flight

// A page that receives tokens: rows [kept, kept + n) of page `to`, from the packed
// tokens first .. first + n - 1, the first of them at `position`.  The rows before
// them are there already, or are copied from page `from`.
struct AppendUnit {
  int first, n, position, kept, to, from;
};

// Unit u.  Sequence b has the units from offsets[b] / page + 2 b on: n tokens touch at
// most (n - 2) / page + 2 pages, and the next sequence starts at least n / page + 2
// further.  Whatever the offsets hold, all indexes stay in range.
__device__ __forceinline__ bool append_unit(const AppendArgs& a, int u, AppendUnit& out) {
  const int lane = threadIdx.x & 31;
  int b = u, begin = u, n = 1, j = 0;
  if (a.offsets) {
    const auto at = [&](int i) { return min(max(__ldg(a.offsets + i), 0), a.tokens); };
    b = 0;
    for (int left = a.sequences; left > 1;) {         // 32 probes a round
      const int step = (left + 31) / 32, i = lane * step;
      const bool before = i < left && at(b + i) / a.page + 2 * (b + i) <= u;
      const int k = max(__popc(__ballot_sync(0xffffffffu, before)) - 1, 0);
      b += k * step;
      left = min(step, left - k * step);
    }
    begin = at(b);
    n = max(at(b + 1) - begin, 0);
    j = u - (begin / a.page + 2 * b);
    if (j < 0) return false;
  }
  constexpr int kMost = 1 << 30;
  const int length = __ldg(a.lengths + b), past = min(max(length, 0), kMost);
  const int column = past / a.page + j;
  if (n == 0 || column > (past + n - 1) / a.page) return false;
  const int low = max(past, column * a.page);
  const int high = (int)min((int64_t)past + n, ((int64_t)column + 1) * a.page);
  out.first = begin + (low - past);
  out.n = high - low;
  out.position = low;
  out.kept = low - column * a.page;
  out.to = -1;
  int error = GRS_OK;
  if (length != past || column >= a.columns) {
    error = GRS_ERR_LENGTH;
  } else {
    out.to = __ldg(a.table + (int64_t)b * a.t_s + column);
    if (out.to < 0 || out.to >= a.pages) out.to = -1, error = GRS_ERR_BAD_PAGE;
  }
  out.from = out.to;
  if (out.kept && a.source && out.to >= 0) {
    out.from = __ldg(a.source + (int64_t)b * a.source_s + column);
    if (out.from < 0 || out.from >= a.pages) out.from = -1, error = GRS_ERR_BAD_PAGE;
  }
  if (error != GRS_OK && threadIdx.x == 0) set_status(a.status, error);
  return true;
}

// A lane's walk over the pieces of consecutive rows.
struct PieceWalk {
  int row, piece;
  __device__ __forceinline__ PieceWalk(int start, int per_row)
      : row(start / per_row), piece(start % per_row) {}
  __device__ __forceinline__ void step(int by, int per_row) {
    for (piece += by; piece >= per_row; piece -= per_row) ++row;
  }
};

// The scale of one head's page, and its kept rows under that scale.  A warp.
template <typename T, int kVec>
__device__ __forceinline__ float append_scale(const AppendArgs& a, const AppendUnit& unit,
                                              const T* rows, int64_t stride, float most,
                                              uint8_t* cache, float* scale) {
  using Codes = RotaryPiece<uint8_t, kVec>;
  const int lane = threadIdx.x & 31, pieces = a.width / kVec;
  float amax = 0.f;
  PieceWalk w(lane, pieces);
  while (w.row < unit.n) {
    RotaryPiece<T, kVec> x[AP_AHEAD];
#pragma unroll
    for (int j = 0; j < AP_AHEAD; ++j) {
      x[j] = {};
      if (w.row >= unit.n) continue;
      x[j] = *reinterpret_cast<const RotaryPiece<T, kVec>*>(rows + w.row * stride + w.piece * kVec);
      w.step(32, pieces);
    }
#pragma unroll
    for (int j = 0; j < AP_AHEAD; ++j)
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float y = fabsf(to_float(x[j].e[i]));
        if (y <= 3.402823466e38f) amax = fmaxf(amax, y);
      }
  }
  const float need = e4m3_scale(warp_max(amax) * most);
  if (!unit.kept || unit.from < 0) {
    if (lane == 0) scale[unit.to * a.s_sp] = need;
    return need;
  }
  const float before = scale[unit.from * a.s_sp], now = fmaxf(before, need);
  if (now != before || unit.from != unit.to) {
    const float ratio = before / now;
    const uint8_t* from = cache + (int64_t)unit.from * a.c_sp;
    uint8_t* to = cache + (int64_t)unit.to * a.c_sp;
    PieceWalk c(lane, pieces);
    while (c.row < unit.kept) {
      Codes x[AP_AHEAD];
      int64_t at[AP_AHEAD];
#pragma unroll
      for (int j = 0; j < AP_AHEAD; ++j) {
        at[j] = -1;
        if (c.row >= unit.kept) continue;
        at[j] = c.row * a.c_st + c.piece * kVec;
        x[j] = *reinterpret_cast<const Codes*>(from + at[j]);
        c.step(32, pieces);
      }
#pragma unroll
      for (int j = 0; j < AP_AHEAD; ++j) {
        if (at[j] < 0) continue;
        if (ratio != 1.f) {
#pragma unroll
          for (int i = 0; i < kVec; ++i) x[j].e[i] = to_e4m3(from_e4m3(x[j].e[i]) * ratio);
        }
        *reinterpret_cast<Codes*>(to + at[j]) = x[j];
      }
    }
  }
  __syncwarp();                             // every lane has read the old scale
  if (lane == 0) scale[unit.to * a.s_sp] = now;
  return now;
}

// One CTA per page that receives tokens and heads_each K/V heads with their query
// heads.  8-bit pages: a warp per head takes the largest value of the page's new
// rows (as they come: the scale does not hang on the rotation's rounding, a pair's
// length bounds what it can become) and moves the rows that are there to the new
// scale.  Then all threads turn, convert and write the new rows, with a table of
// the rows' (cos, sin) in shared memory.
template <typename T, int kVec, bool kInter, bool kCodes>
__global__ void __launch_bounds__(AP_THREADS) append_kernel(AppendArgs a) {
  using Units = RotaryUnits<kVec, kInter>;
  using Piece = RotaryPiece<T, kVec>;
  using Store = typename std::conditional<kCodes, uint8_t, T>::type;
  extern __shared__ float2 ap_turns[];
  float* inverse = reinterpret_cast<float*>(ap_turns + a.rows * a.pairs);   // [2][heads_each]
  const int warp = threadIdx.x >> 5;
  const int h0 = blockIdx.y * a.heads_each, nh = min(a.heads_each, a.kv_heads - h0);
  const int nq = a.q ? nh * a.group : 0;

  if ((int)blockIdx.x >= a.units) {         // rows of no sequence
    const int begin = min(max(__ldg(a.offsets), 0), a.tokens);
    const int end = min(max(__ldg(a.offsets + a.sequences), begin), a.tokens);
    const int rest = begin + a.tokens - end, all = nq * a.width;
    for (int r = blockIdx.x - a.units; r < rest; r += gridDim.x - a.units) {
      T* row = static_cast<T*>(a.qo) + (int64_t)(r < begin ? r : end + r - begin) * a.qo_st +
               (int64_t)h0 * a.group * a.qo_sh;
      for (int i = threadIdx.x; i < all; i += AP_THREADS)
        row[i / a.width * a.qo_sh + i % a.width] = from_float<T>(0.f);
    }
    return;
  }
  AppendUnit unit;
  if (!append_unit(a, blockIdx.x, unit)) return;
  const auto cache = [&](bool value) { return static_cast<Store*>(value ? a.vc : a.kc); };
  const auto fresh = [&](bool value) { return static_cast<const T*>(value ? a.v : a.k); };

  if (unit.to >= 0) {
    if constexpr (kCodes) {
      for (int task = warp; task < 2 * nh; task += AP_THREADS / 32) {
        const bool which = task >= nh;
        const int h = h0 + (which ? task - nh : task);
        const int64_t st = which ? a.v_st : a.k_st, sh = which ? a.v_sh : a.k_sh;
        const float s = append_scale<T, kVec>(
            a, unit, fresh(which) + unit.first * st + h * sh, st, which ? 1.f : a.key_most,
            cache(which) + h * a.c_sh, (which ? a.vs : a.ks) + h);
        if ((threadIdx.x & 31) == 0) inverse[task] = 1.f / s;
      }
    } else if (unit.kept && unit.from >= 0 && unit.from != unit.to) {
      const int pieces = a.width / kVec;
      for (int task = warp; task < 2 * nh * unit.kept; task += AP_THREADS / 32) {
        const int head = task / unit.kept, row = task - head * unit.kept;
        const bool which = head >= nh;
        const int64_t at = row * a.c_st + (h0 + (which ? head - nh : head)) * a.c_sh;
        for (int p = threadIdx.x & 31; p < pieces; p += 32)
          *reinterpret_cast<Piece*>(cache(which) + (int64_t)unit.to * a.c_sp + at + p * kVec) =
              *reinterpret_cast<const Piece*>(cache(which) + (int64_t)unit.from * a.c_sp + at +
                                              p * kVec);
      }
    }
  }

  const int units = Units::count(a.width, a.pairs), each = AP_THREADS / units;
  const int all = nq + (unit.to >= 0 ? 2 * nh : 0);
  const bool works = all > 0 && threadIdx.x < each * units;
  const Units place(threadIdx.x % units, a.pairs);
  for (int r0 = 0; r0 < unit.n; r0 += a.rows) {
    const int n = min(a.rows, unit.n - r0);
    __syncthreads();                        // the scales are known, the last table is read
    for (int i = threadIdx.x; i < n * a.pairs; i += AP_THREADS) {
      const int row = r0 + i / a.pairs, at = unit.first + row;
      int64_t p = unit.position + row;
      if (a.positions)
        p = a.wide ? static_cast<const int64_t*>(a.positions)[at]
                   : static_cast<const int32_t*>(a.positions)[at];
      const float2 t = rotary_cos_sin(rotary_phase(p, rotary_step(a.freq[i % a.pairs])));
      ap_turns[i] = make_float2(t.x * a.magnitude, t.y * a.magnitude);
    }
    __syncthreads();
    if (!works) continue;
    int head = threadIdx.x / units % all, row = threadIdx.x / units / all;
    while (row < n) {
      Piece x[AP_AHEAD], y[AP_AHEAD];
      int heads[AP_AHEAD], rows[AP_AHEAD];
#pragma unroll
      for (int j = 0; j < AP_AHEAD; ++j) {
        heads[j] = -1;
        if (row >= n) continue;
        heads[j] = head;
        rows[j] = row;
        const int64_t at = unit.first + r0 + row;
        const T* from = head < nq        ? static_cast<const T*>(a.q) + at * a.q_st +
                                               (int64_t)(h0 * a.group + head) * a.q_sh
                        : head < nq + nh ? fresh(false) + at * a.k_st + (h0 + head - nq) * a.k_sh
                                         : fresh(true) + at * a.v_st + (h0 + head - nq - nh) * a.v_sh;
        x[j] = *reinterpret_cast<const Piece*>(from + place.a);
        if (place.two()) y[j] = *reinterpret_cast<const Piece*>(from + place.b);
        for (head += each; head >= all; head -= all) ++row;
      }
#pragma unroll
      for (int j = 0; j < AP_AHEAD; ++j) {
        if (heads[j] < 0) continue;
        const bool query = heads[j] < nq, value = heads[j] >= nq + nh;
        float u[kVec], w[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          u[i] = to_float(x[j].e[i]);
          w[i] = Units::kTwo && place.pair >= 0 ? to_float(y[j].e[i]) : 0.f;
        }
        if (!value && place.pair >= 0)
          rotary_turn<T, kVec, kInter>(ap_turns + rows[j] * a.pairs + place.pair, u, w);
        if (query || !kCodes) {
          T* to;
          if (query)
            to = static_cast<T*>(a.qo) + (int64_t)(unit.first + r0 + rows[j]) * a.qo_st +
                 (int64_t)(h0 * a.group + heads[j]) * a.qo_sh;
          else
            to = reinterpret_cast<T*>(cache(value)) + (int64_t)unit.to * a.c_sp +
                 (int64_t)(unit.kept + r0 + rows[j]) * a.c_st +
                 (h0 + heads[j] - nq - (value ? nh : 0)) * a.c_sh;
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            x[j].e[i] = from_float<T>(u[i]);
            y[j].e[i] = from_float<T>(w[i]);
          }
          *reinterpret_cast<Piece*>(to + place.a) = x[j];
          if (place.two()) *reinterpret_cast<Piece*>(to + place.b) = y[j];
        } else {
          using Codes = RotaryPiece<uint8_t, kVec>;
          const int h = heads[j] - nq - (value ? nh : 0);
          const float inv = inverse[heads[j] - nq];
          uint8_t* to = reinterpret_cast<uint8_t*>(cache(value)) + (int64_t)unit.to * a.c_sp +
                        (int64_t)(unit.kept + r0 + rows[j]) * a.c_st + (h0 + h) * a.c_sh;
          Codes c, d;
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            c.e[i] = to_e4m3(u[i] * inv);
            d.e[i] = to_e4m3(w[i] * inv);
          }
          *reinterpret_cast<Codes*>(to + place.a) = c;
          if (place.two()) *reinterpret_cast<Codes*>(to + place.b) = d;
        }
      }
    }
  }
}

template <typename T>
static int append_run(AppendArgs a, bool interleaved, cudaStream_t stream) {
  const int e = sizeof(T);
  const bool codes = a.ks != nullptr;
  int alignment = std::min(common_alignment(a.k, a.k_st * e, a.k_sh * e),
                           common_alignment(a.v, a.v_st * e, a.v_sh * e));
  if (a.q)
    alignment = std::min({alignment, common_alignment(a.q, a.q_st * e, a.q_sh * e),
                          common_alignment(a.qo, a.qo_st * e, a.qo_sh * e)});
  const int p = codes ? 1 : e;
  const int cache = std::min(common_alignment(a.kc, a.c_sp * p, a.c_st * p, a.c_sh * p),
                             common_alignment(a.vc));
  alignment = std::min(alignment, cache * (e / p));   // a piece has as many codes as elements
  const int64_t units = a.offsets && a.sequences
                            ? (int64_t)a.tokens / a.page + 2 * (int64_t)a.sequences
                            : a.sequences;
  if (units > INT_MAX - 64) return GRS_ERR_SHAPE;
  a.units = (int)units;
  const int split = (int)std::min<int64_t>(a.kv_heads, std::max<int64_t>(1, 4 * 148 / std::max<int64_t>(1, units)));
  a.heads_each = (a.kv_heads + split - 1) / split;
  a.rows = a.offsets ? std::min(AP_ROWS, a.page) : 1;
  const dim3 grid((unsigned)(units + (a.clear ? 64 : 0)),
                  (a.kv_heads + a.heads_each - 1) / a.heads_each);
  if (grid.y > 65535) return GRS_ERR_SHAPE;
  const int64_t smem = (int64_t)a.rows * a.pairs * sizeof(float2) + 8 * (int64_t)a.heads_each;
  if (smem > 48 * 1024) return GRS_ERR_SHAPE;
  return rotary_dispatch<T>(a.width, a.pairs, interleaved, alignment,
                            [&](auto vec, auto inter) -> int {
    constexpr int kVec = decltype(vec)::value;
    constexpr bool kInter = decltype(inter)::value;
    if (codes)
      append_kernel<T, kVec, kInter, true><<<grid, AP_THREADS, smem, counted(stream)>>>(a);
    else
      append_kernel<T, kVec, kInter, false><<<grid, AP_THREADS, smem, counted(stream)>>>(a);
    GRS_CUDA_CHECK_LAUNCH();
    return GRS_OK;
  });
}

}  // namespace grs

extern "C" int grs_append_tokens(
    int dtype, int cache_dtype, const void* query, int64_t q_st, int64_t q_sh, void* query_out,
    int64_t qo_st, int64_t qo_sh, int clear_rest, const void* key, int64_t k_st, int64_t k_sh,
    const void* value, int64_t v_st, int64_t v_sh, void* key_cache, void* value_cache,
    int64_t c_sp, int64_t c_st, int64_t c_sh, float* key_scale, float* value_scale, int64_t s_sp,
    const int32_t* block_table, int64_t bt_stride, const int32_t* source_table,
    int64_t source_stride, int max_blocks, const int32_t* lengths, const int32_t* offsets,
    const void* positions, int positions_are_i64, const double* frequencies, int pairs,
    int interleaved, double magnitude, int tokens, int sequences, int heads, int kv_heads,
    int head_width, int num_pages, int page_size, int32_t* status, void* stream) {
  using namespace grs;
  constexpr int kMost = 1 << 30;
  const bool codes = cache_dtype == GRS_DTYPE_E4M3;
  if ((dtype != GRS_DTYPE_F32 && dtype != GRS_DTYPE_BF16) || (!codes && cache_dtype != dtype) ||
      tokens < 0 || tokens >= kMost || sequences < 0 || sequences >= kMost || kv_heads <= 0 ||
      kv_heads >= kMost || heads < 0 || heads >= kMost || heads % kv_heads ||
      (query && heads == 0) || head_width <= 0 || head_width > 256 || pairs < 0 ||
      2 * pairs > head_width || !std::isfinite(magnitude) || num_pages < 0 || max_blocks < 0 ||
      page_size <= 0 || page_size >= kMost || (int64_t)max_blocks * page_size >= kMost ||
      (!offsets && tokens != sequences))
    return GRS_ERR_SHAPE;
  if (tokens == 0) return GRS_OK;
  if (!key || !value || (query && !query_out) || (pairs && !frequencies) ||
      (sequences && !lengths) || (max_blocks && sequences && !block_table) ||
      (num_pages && (!key_cache || !value_cache)) ||
      (codes && num_pages && (!key_scale || !value_scale)))
    return GRS_ERR_SHAPE;
  AppendArgs a = {};
  a.q = query; a.q_st = q_st; a.q_sh = q_sh; a.qo = query_out; a.qo_st = qo_st; a.qo_sh = qo_sh;
  a.k = key; a.k_st = k_st; a.k_sh = k_sh; a.v = value; a.v_st = v_st; a.v_sh = v_sh;
  a.kc = key_cache; a.vc = value_cache; a.c_sp = c_sp; a.c_st = c_st; a.c_sh = c_sh;
  a.ks = codes ? key_scale : nullptr; a.vs = codes ? value_scale : nullptr; a.s_sp = s_sp;
  a.table = block_table; a.t_s = bt_stride; a.source = source_table; a.source_s = source_stride;
  a.columns = max_blocks; a.lengths = lengths; a.offsets = offsets;
  a.positions = positions; a.wide = positions_are_i64;
  a.freq = frequencies; a.pairs = pairs; a.magnitude = (float)magnitude;
  // sqrt(2), rounded up: a pair's length over its larger element
  a.key_most = pairs ? (float)std::max(1.0, 1.41421366 * std::fabs(magnitude)) : 1.f;
  a.tokens = tokens; a.sequences = sequences; a.group = heads / kv_heads; a.kv_heads = kv_heads;
  a.width = head_width; a.pages = num_pages; a.page = page_size;
  a.clear = clear_rest && query && offsets; a.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (sequences == 0 && !a.clear) return GRS_OK;
  return dtype == GRS_DTYPE_F32 ? append_run<float>(a, interleaved != 0, s)
                                : append_run<__nv_bfloat16>(a, interleaved != 0, s);
}
