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
  const int32_t* table; int64_t t_s; const int32_t* source; int64_t source_s; int source_columns, columns;
  const int32_t* lengths; const int32_t* offsets;     // offsets null: a token per sequence
  const void* positions; int wide;                    // int32 or int64 [tokens], or null
  const double* freq; int pairs; float magnitude, key_most;
  int tokens, sequences, group, kv_heads, width, pages, page;
  int units, heads_each, rows, code_bytes, clear;
  int32_t* status;
  const int32_t* shut;                                // or null: nothing is written while set
};

// Threads of a CTA: at least one for each unit of a head.
constexpr int append_threads(int vec) { return vec == 1 ? 256 : 128; }

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
  out.to = out.from = -1;
  if (a.shut && *a.shut != 0) return true;            // queries are turned all the same
  int error = GRS_OK;
  if (length != past || column >= a.columns) {
    error = GRS_ERR_LENGTH;
  } else {
    out.to = __ldg(a.table + (int64_t)b * a.t_s + column);
    if (out.to < 0 || out.to >= a.pages) out.to = -1, error = GRS_ERR_BAD_PAGE;
  }
  out.from = out.to;
  if (out.kept && a.source && out.to >= 0) {
    out.from = column < a.source_columns
                   ? __ldg(a.source + (int64_t)b * a.source_s + column) : -1;
    if (out.from < 0 || out.from >= a.pages) out.from = -1, error = GRS_ERR_BAD_PAGE;
  }
  if (error != GRS_OK && threadIdx.x == 0) set_status(a.status, error);
  return true;
}

// The kept rows of one head's page, times `ratio` (1: copied), from one page to another or
// in place: pieces of kBytes codes, whole rows side by side in a warp's lanes, kHold pieces
// of a lane at once.
template <int kBytes>
struct KeptCodes {
  using Word = typename std::conditional<
      kBytes == 16, uint4, typename std::conditional<kBytes == 8, uint2, uint8_t>::type>::type;
  static constexpr int kHold = 4;
  Word x[kHold];
  int64_t at;                               // of the first piece
  int row, by;                              // first row, rows of a step
  __device__ __forceinline__ KeptCodes(int64_t stride, int width, int part) {
    const int lane = threadIdx.x & 31, pieces = min(width / kBytes - 32 * part, 32);
    row = lane / pieces;
    by = 32 / pieces;
    at = row * stride + (lane - row * pieces + 32 * part) * kBytes;
    if (row >= by) row = 1 << 30;           // lanes that are left over
  }
  __device__ __forceinline__ void load(const uint8_t* from, int64_t stride, int rows, int round) {
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      const int step = (round * kHold + j) * by;
      if (row + step < rows) x[j] = *reinterpret_cast<const Word*>(from + at + step * stride);
    }
  }
  __device__ __forceinline__ void store(uint8_t* to, int64_t stride, int rows, int round,
                                        float ratio) {
    const bool halves = (__float_as_uint(ratio) & 0x7fffffu) == 0 && ratio <= 1.f;
    const __half2 scale = __float2half2_rn(ratio);
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      const int step = (round * kHold + j) * by;
      if (row + step >= rows) continue;
      if (ratio != 1.f) {
        if constexpr (kBytes == 1) {
          x[j] = to_e4m3(from_e4m3(x[j]) * ratio);
        } else {
          uint32_t* v = reinterpret_cast<uint32_t*>(&x[j]);
#pragma unroll
          for (int k = 0; k < kBytes / 4; ++k)
            v[k] = halves ? e4m3x2_times(v[k], scale) | e4m3x2_times(v[k] >> 16, scale) << 16
                          : e4m3x4_times(v[k], ratio);
        }
      }
      *reinterpret_cast<Word*>(to + at + step * stride) = x[j];
    }
  }
  static __device__ __forceinline__ void move(const uint8_t* from, uint8_t* to, int64_t stride,
                                              int rows, int width, float ratio) {
    for (int part = 0; part * 32 * kBytes < width; ++part) {
      KeptCodes codes(stride, width, part);
      for (int round = 0; round * kHold * codes.by < rows; ++round) {
        codes.load(from, stride, rows, round);
        codes.store(to, stride, rows, round, ratio);
      }
    }
  }
};
// Out of line: it is rare, or short, beside the code around it.
static __device__ __noinline__ void append_move(const uint8_t* from, uint8_t* to, int64_t stride, int rows,
                                         int width, int bytes, float ratio) {
  if (bytes == 16)
    KeptCodes<16>::move(from, to, stride, rows, width, ratio);
  else if (bytes == 8)
    KeptCodes<8>::move(from, to, stride, rows, width, ratio);
  else
    KeptCodes<1>::move(from, to, stride, rows, width, ratio);
}

// A lane's walk over the units of consecutive rows at `at`: whole rows side by side in
// the warp, or a row in several rounds.  Units of 32 and less keep their lanes, whose
// place then changes by whole strides only.
template <typename T, int kVec, bool kInter>
struct RowWalk {
  using Units = RotaryUnits<kVec, kInter>;
  T* at;                                    // the row
  int64_t stride;                           // of a step
  int row, index, by;                       // unit's index in the row; rows of a step, or 0
  Units unit;
  __device__ __forceinline__ RowWalk(T* base, int64_t st, int units, int pairs)
      : unit((int)(threadIdx.x & 31) % min(units, 32), pairs) {
    const int lane = threadIdx.x & 31;
    by = 32 / units;
    row = by ? lane / units : 0;
    index = by ? 0 : lane;
    if (row >= max(by, 1)) row = 1 << 30;   // lanes that are left over
    at = base + (row < (1 << 30) ? row * st : 0);
    stride = max(by, 1) * st;
  }
  __device__ __forceinline__ bool inside(int n, int units) const {
    return row < n && index < units;
  }
  __device__ __forceinline__ void step(int units, int pairs) {
    if (by) {
      row += by;
      at += stride;
    } else {
      index += 32;
      if (index >= (units + 31) / 32 * 32 + (int)(threadIdx.x & 31)) {
        index = threadIdx.x & 31;
        ++row;
        at += stride;
      }
      unit = Units(min(index, units - 1), pairs);
    }
  }
  static __device__ __forceinline__ int rounds(int n, int units) {
    return units <= 32 ? (n + 32 / units - 1) / (32 / units) : n * ((units + 31) / 32);
  }
};

// The new rows of one head's page, key or value, by a warp: kHold units of a lane at
// once.  8-bit pages: the largest value of all of them first, which gives the scale.  Rows
// that fit kHold rounds (up to 16 of 128 bf16 elements) stay in registers until it is known;
// more are read twice (ragged prompts into pages of 16 / 32 / 64 tokens: 80 / 92 / 96 us).
template <typename T, int kVec, bool kInter, bool kCodes, int kHold>
struct AppendHead {
  using Units = RotaryUnits<kVec, kInter>;
  using Piece = RotaryPiece<T, kVec>;
  using Store = typename std::conditional<kCodes, uint8_t, T>::type;
  Piece x[kHold], y[kHold];

  __device__ __forceinline__ void fetch(RowWalk<const T, kVec, kInter>& walk, int n, int units,
                                        int pairs) {
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      x[j].clear();
      y[j].clear();
      if (walk.inside(n, units)) {
        x[j].load(walk.at + walk.unit.a);
        if (walk.unit.two()) y[j].load(walk.at + walk.unit.b);
      }
      walk.step(units, pairs);
    }
  }
  // The largest absolute value held, as its bits; what is not finite is larger than
  // any number, or with `finite` left out.
  __device__ __forceinline__ uint32_t largest(bool finite) const {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      top = max(top, x[j].largest(finite));
      if constexpr (Units::kTwo) top = max(top, y[j].largest(finite));
    }
    return top;
  }
  __device__ __forceinline__ void store(RowWalk<Store, kVec, kInter>& walk, int n, int units,
                                        int pairs, const float* table, float inverse) {
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      if (walk.inside(n, units)) {
        const Units& unit = walk.unit;
        float u[kVec], v[kVec] = {};
        x[j].get(u);
        if constexpr (Units::kTwo) y[j].get(v);
        if (table && unit.pair >= 0) {
          RotaryTurns<kVec, kInter> turns;
          turns.get(table + 2 * walk.row * pairs, unit.pair, pairs);
          turns.turn(u, v);
        }
        if constexpr (kCodes) {
          e4m3_store<kVec>(walk.at + unit.a, u, inverse);
          if (unit.two()) e4m3_store<kVec>(walk.at + unit.b, v, inverse);
        } else {
          x[j].set(u);
          x[j].store(walk.at + unit.a);
          if (unit.two()) {
            y[j].set(v);
            y[j].store(walk.at + unit.b);
          }
        }
      }
      walk.step(units, pairs);
    }
  }
};

// One CTA per page that receives tokens and heads_each K/V heads with their query
// heads.  A warp per key or value head: with 8-bit pages it finds the scale (on the
// values as they come, not on the rotation's rounding: a pair's length bounds what it
// becomes) and moves the rows that are there to it; then it turns, converts and writes
// the new rows.  All threads turn the queries.  A table of the rows' (cos, sin) in
// shared memory serves all of them.  16384 tokens, 32/8 heads of 128, into bf16 pages:
// 72 us = 5.6 TB/s, by HBM; 13930 tokens of 16 prompts into 8-bit pages 77 us = 4.4 TB/s,
// by latency: the rows wait in registers for their scale, which leaves 16 warps an SM
// (12 of 170 registers 102 us, 20 of 96 spill, 123).
template <typename T, int kVec, bool kInter, bool kCodes>
__global__ void __launch_bounds__(append_threads(kVec), kVec == 1 ? 2 : 4)
    append_kernel(AppendArgs a) {
  constexpr int kThreads = append_threads(kVec);
  using Units = RotaryUnits<kVec, kInter>;
  using From = RowWalk<const T, kVec, kInter>;
  using Store = typename std::conditional<kCodes, uint8_t, T>::type;
  constexpr int kHold = Units::kTwo ? 4 : 8;
  extern __shared__ __align__(16) float ap_turns[];
  float* inverses = ap_turns + 2 * a.rows * a.pairs;      // [2 heads_each]
  float* ratios = inverses + 2 * a.heads_each;            // [2 heads_each]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h0 = blockIdx.y * a.heads_each, nh = min(a.heads_each, a.kv_heads - h0);
  const int q0 = h0 * a.group, nq = a.q ? nh * a.group : 0;

  if ((int)blockIdx.x >= a.units) {         // query rows of no sequence
    const int begin = min(max(__ldg(a.offsets), 0), a.tokens);
    const int end = min(max(__ldg(a.offsets + a.sequences), begin), a.tokens);
    const int rest = begin + a.tokens - end;
    for (int r = blockIdx.x - a.units; r < rest; r += gridDim.x - a.units) {
      T* row = static_cast<T*>(a.qo) + (int64_t)(r < begin ? r : end + r - begin) * a.qo_st +
               q0 * a.qo_sh;
      for (int h = warp; h < nq; h += kThreads / 32)
        for (int i = lane; i < a.width; i += 32) row[h * a.qo_sh + i] = from_float<T>(0.f);
    }
    return;
  }
  AppendUnit unit;
  if (!append_unit(a, blockIdx.x, unit)) return;

  // key heads, then value heads, in turn by the warps
  const int units = Units::count(a.width, a.pairs), rounds = From::rounds(unit.n, units);
  const int tasks = unit.to >= 0 ? 2 * nh : 0, blocks = (unit.n + a.rows - 1) / a.rows;
  const bool held = blocks == 1 && rounds <= kHold;       // a task's rows in registers
  const auto stride_of = [&](int task) { return task >= nh ? a.v_st : a.k_st; };
  const auto rows_of = [&](int task) {
    const bool value = task >= nh;
    return static_cast<const T*>(value ? a.v : a.k) + unit.first * stride_of(task) +
           (h0 + (value ? task - nh : task)) * (value ? a.v_sh : a.k_sh);
  };
  const auto cache_of = [&](int task, int page) {
    const bool value = task >= nh;
    return static_cast<Store*>(value ? a.vc : a.kc) + (int64_t)page * a.c_sp +
           (h0 + (value ? task - nh : task)) * a.c_sh;
  };
  AppendHead<T, kVec, kInter, kCodes, kHold> head;
  const auto fetch = [&](int task) {
    From walk(rows_of(task), stride_of(task), units, a.pairs);
    head.fetch(walk, unit.n, units, a.pairs);
  };
  // 8-bit pages: the scale of a task's page and its inverse; what moves the kept rows to it
  // (-1: they stay) is left for the end, when nothing else is held
  const bool moved = unit.kept && unit.from >= 0;
  const auto scale = [&](int task) {
    if constexpr (!kCodes) return 1.f;
    const bool value = task >= nh;
    float* scales = (value ? a.vs : a.ks) + h0 + (value ? task - nh : task);
    const float before = moved ? scales[unit.from * a.s_sp] : 0.f;
    const auto largest = [&](bool finite) {
      uint32_t top = 0;
      if (held) {
        top = head.largest(finite);
      } else {
        From walk(rows_of(task), stride_of(task), units, a.pairs);
        for (int r = 0; r < rounds; r += kHold) {
          head.fetch(walk, unit.n, units, a.pairs);
          top = max(top, head.largest(finite));
        }
      }
      return __reduce_max_sync(0xffffffffu, top);
    };
    uint32_t top = largest(false);
    if (top >= 0x7f800000u) top = largest(true);
    const float now = fmaxf(before, e4m3_scale(__uint_as_float(top) * (value ? 1.f : a.key_most)));
    __syncwarp();                           // every lane has read the old scale
    if (lane == 0) {
      scales[unit.to * a.s_sp] = now;
      ratios[task] = moved && (now != before || unit.from != unit.to) ? before / now : -1.f;
    }
    return 1.f / now;
  };
  if constexpr (!kCodes) {
    if (moved && unit.from != unit.to) {
      const int pieces = a.width / kVec, count = unit.kept * pieces;
      for (int task = warp; task < tasks; task += kThreads / 32)
        for (int i = lane; i < count; i += 32) {
          const int64_t at = i / pieces * a.c_st + i % pieces * kVec;
          RotaryPiece<T, kVec> x;
          x.load(reinterpret_cast<const T*>(cache_of(task, unit.from)) + at);
          x.store(reinterpret_cast<T*>(cache_of(task, unit.to)) + at);
        }
    }
  }
  if (kCodes && held && warp < tasks) fetch(warp);    // under the table
  if (kCodes && !held)
    for (int task = warp; task < tasks; task += kThreads / 32) {
      const float inverse = scale(task);
      if (lane == 0) inverses[task] = inverse;
    }

  for (int block = 0; block < blocks; ++block) {          // rows of a table
    const int r0 = block * a.rows, n = min(a.rows, unit.n - r0);
    if (block) __syncthreads();             // the last table is read
    rotary_table<kVec, kInter, kThreads>(
        ap_turns, a.freq, a.pairs, a.magnitude, n, [&](int row) -> int64_t {
          if (!a.positions) return unit.position + r0 + row;
          return a.wide ? static_cast<const int64_t*>(a.positions)[unit.first + r0 + row]
                        : static_cast<const int32_t*>(a.positions)[unit.first + r0 + row];
        });
    __syncthreads();
    const int64_t first = unit.first + r0;
    if constexpr (!kCodes) {
      if (tasks) {
        const int64_t at = (int64_t)unit.to * a.c_sp + (unit.kept + r0) * a.c_st + h0 * a.c_sh;
        rotary_rows_apart<T, kVec, kInter, kThreads>(
            ap_turns, a.pairs, a.width, n, nh,
            static_cast<const T*>(a.k) + first * a.k_st + h0 * a.k_sh, a.k_st, a.k_sh,
            static_cast<T*>(a.kc) + at, a.c_st, a.c_sh);
        rotary_rows_apart<T, kVec, kInter, kThreads>(
            ap_turns, 0, a.width, n, nh,
            static_cast<const T*>(a.v) + first * a.v_st + h0 * a.v_sh, a.v_st, a.v_sh,
            static_cast<T*>(a.vc) + at, a.c_st, a.c_sh);
      }
    }
    for (int task = warp; kCodes && task < tasks; task += kThreads / 32) {
      float inverse = 1.f;
      if (held) {
        if (task != warp) fetch(task);
        inverse = scale(task);
      } else {
        inverse = inverses[task];
      }
      From there(rows_of(task) + r0 * stride_of(task), stride_of(task), units, a.pairs);
      RowWalk<Store, kVec, kInter> walk(cache_of(task, unit.to) + (unit.kept + r0) * a.c_st, a.c_st,
                                        units, a.pairs);
      for (int r = From::rounds(n, units); r > 0; r -= kHold) {
        if (!held) head.fetch(there, n, units, a.pairs);
        head.store(walk, n, units, a.pairs, task >= nh ? nullptr : ap_turns, inverse);
      }
    }
    if (nq) {
      rotary_rows_apart<T, kVec, kInter, kThreads>(
          ap_turns, a.pairs, a.width, n, nq,
          static_cast<const T*>(a.q) + first * a.q_st + q0 * a.q_sh, a.q_st, a.q_sh,
          static_cast<T*>(a.qo) + first * a.qo_st + q0 * a.qo_sh, a.qo_st, a.qo_sh);
    }
  }
  if (kCodes && moved)
    for (int task = warp; task < tasks; task += kThreads / 32) {
      __syncwarp();
      if (ratios[task] != -1.f)
        append_move(reinterpret_cast<const uint8_t*>(cache_of(task, unit.from)),
                    reinterpret_cast<uint8_t*>(cache_of(task, unit.to)), a.c_st, unit.kept, a.width,
                    a.code_bytes, ratios[task]);
    }
}

// One token per sequence: a CTA per sequence and heads_each K/V heads with their query
// heads.  A thread keeps one place in the head and takes every slots-th of the key,
// value and query heads; the first rounds are fetched before anything else is known,
// and the rows of the last page that are to be copied under the table of (cos, sin):
// the call is a chain of latencies, not of bytes.  1000 forked tokens, 32/8 heads of 128,
// into 8-bit pages: 22 us, of which 52 MB are 8; five tokens 3 us.
template <typename T, int kVec, bool kInter, bool kCodes>
__global__ void __launch_bounds__(append_threads(kVec), kVec == 1 ? 2 : 4)
    append_one_kernel(AppendArgs a) {
  constexpr int kThreads = append_threads(kVec);
  using Units = RotaryUnits<kVec, kInter>;
  using Piece = RotaryPiece<T, kVec>;
  using Store = typename std::conditional<kCodes, uint8_t, T>::type;
  constexpr int kHeld = Units::kTwo ? 3 : 6;
  extern __shared__ __align__(16) float ap_turns[];
  uint32_t* tops = reinterpret_cast<uint32_t*>(ap_turns + 2 * a.pairs);   // [2 heads_each]
  float* inverses = reinterpret_cast<float*>(tops + 2 * a.heads_each);    // [2 heads_each]
  float* ratios = inverses + 2 * a.heads_each;                            // [2 heads_each]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x;
  const int h0 = blockIdx.y * a.heads_each, nh = min(a.heads_each, a.kv_heads - h0);
  const int all = 2 * nh + (a.q ? nh * a.group : 0);
  const int units = Units::count(a.width, a.pairs), slots = kThreads / units;
  const int slot = threadIdx.x / units;
  const Units unit(threadIdx.x - slot * units, a.pairs);
  const auto head_at = [&](int i) {         // key heads, value heads, query heads
    return i < nh       ? static_cast<const T*>(a.k) + b * a.k_st + (h0 + i) * a.k_sh
           : i < 2 * nh ? static_cast<const T*>(a.v) + b * a.v_st + (h0 + i - nh) * a.v_sh
                        : static_cast<const T*>(a.q) + b * a.q_st +
                              (h0 * a.group + i - 2 * nh) * a.q_sh;
  };
  Piece x[kHeld], y[kHeld];
  const auto fetch = [&](int i, Piece& u, Piece& v) {
    if (slot >= slots || i >= all) return;
    const T* at = head_at(i);
    u.load(at + unit.a);
    if (unit.two()) v.load(at + unit.b);
  };
#pragma unroll
  for (int r = 0; r < kHeld; ++r) fetch(slot + r * slots, x[r], y[r]);
  for (int i = threadIdx.x; i < 2 * nh; i += kThreads) tops[i] = 0;
  AppendUnit page;
  append_unit(a, b, page);
  const bool kept = page.to >= 0 && page.kept && page.from >= 0, copied = kept && page.from != page.to;

  // this warp's first head of the kept rows
  const auto cache_of = [&](int task, int at) {
    return static_cast<Store*>(task >= nh ? a.vc : a.kc) + (int64_t)at * a.c_sp +
           (h0 + (task >= nh ? task - nh : task)) * a.c_sh;
  };
  const auto scale_of = [&](int task) {
    return (task >= nh ? a.vs : a.ks) + h0 + (task >= nh ? task - nh : task);
  };
  float before = 0.f;
  const bool ahead = kCodes && copied && a.code_bytes == 16;
  KeptCodes<16> codes(a.c_st, ahead ? a.width : 16, 0);
  if (warp < 2 * nh) {
    if (kCodes && kept) before = scale_of(warp)[page.from * a.s_sp];
    if (ahead)
      codes.load(reinterpret_cast<const uint8_t*>(cache_of(warp, page.from)), a.c_st, page.kept, 0);
  }
  rotary_table<kVec, kInter, kThreads>(ap_turns, a.freq, a.pairs, a.magnitude, 1, [&](int) -> int64_t {
    if (!a.positions) return page.position;
    return a.wide ? static_cast<const int64_t*>(a.positions)[b]
                  : static_cast<const int32_t*>(a.positions)[b];
  });
  __syncthreads();
  RotaryTurns<kVec, kInter> turns;
  if (unit.pair >= 0) turns.get(ap_turns, unit.pair, a.pairs);
  if constexpr (kCodes) {
    const auto top_of = [&](int i, const Piece& u, const Piece& v) {
      if (slot >= slots || i >= 2 * nh) return;
      const auto both = [&](bool finite) {
        const uint32_t top = u.largest(finite);
        return unit.two() ? max(top, v.largest(finite)) : top;
      };
      uint32_t top = both(false);
      if (top >= 0x7f800000u) top = both(true);   // not finite
      atomicMax(&tops[i], top);
    };
#pragma unroll
    for (int r = 0; r < kHeld; ++r) top_of(slot + r * slots, x[r], y[r]);
    for (int i = slot + kHeld * slots; i < 2 * nh; i += slots) {
      Piece u, v;
      fetch(i, u, v);
      top_of(i, u, v);
    }
    __syncthreads();
  }
  for (int task = warp; task < 2 * nh && page.to >= 0; task += kThreads / 32) {
    if constexpr (kCodes) {
      float* scale = scale_of(task);
      if (kept && task != warp) before = scale[page.from * a.s_sp];
      const float need = e4m3_scale(__uint_as_float(tops[task]) *
                                    (task >= nh ? 1.f : a.key_most));
      const float now = fmaxf(before, need);
      const float ratio = before / now;
      if (ahead) {
        const uint8_t* from = reinterpret_cast<const uint8_t*>(cache_of(task, page.from));
        uint8_t* to = reinterpret_cast<uint8_t*>(cache_of(task, page.to));
        for (int round = 0; round * codes.kHold * codes.by < page.kept; ++round) {
          if (task != warp || round) codes.load(from, a.c_st, page.kept, round);
          codes.store(to, a.c_st, page.kept, round, ratio);
        }
      }
      __syncwarp();                         // every lane has read the old scale
      if (lane == 0) {
        scale[page.to * a.s_sp] = now;
        inverses[task] = 1.f / now;
        ratios[task] = kept && !ahead && (now != before || copied) ? ratio : -1.f;
      }
    } else if (copied) {
      const int each = a.width / kVec, n = page.kept * each;
      const T* from = reinterpret_cast<const T*>(cache_of(task, page.from));
      T* to = reinterpret_cast<T*>(cache_of(task, page.to));
      constexpr int kCopies = 4;
      for (int i0 = lane; i0 < n; i0 += 32 * kCopies) {
        Piece z[kCopies];
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
          const int i = i0 + 32 * j;
          if (i < n) z[j].load(from + i / each * a.c_st + i % each * kVec);
        }
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
          const int i = i0 + 32 * j;
          if (i < n) z[j].store(to + i / each * a.c_st + i % each * kVec);
        }
      }
    }
  }
  const auto write = [&](int i, Piece& u, Piece& v, bool queries) {
    if (slot >= slots || i >= all || (i >= 2 * nh) != queries) return;
    float p[kVec], q[kVec] = {};
    u.get(p);
    if constexpr (Units::kTwo) v.get(q);
    if (unit.pair >= 0 && (i < nh || queries)) turns.turn(p, q);
    if (queries || !kCodes) {
      T* to = queries ? static_cast<T*>(a.qo) + b * a.qo_st + (h0 * a.group + i - 2 * nh) * a.qo_sh
                      : reinterpret_cast<T*>(cache_of(i, page.to)) + page.kept * a.c_st;
      u.set(p);
      u.store(to + unit.a);
      if (unit.two()) {
        v.set(q);
        v.store(to + unit.b);
      }
    } else {
      uint8_t* to = reinterpret_cast<uint8_t*>(cache_of(i, page.to)) + page.kept * a.c_st;
      e4m3_store<kVec>(to + unit.a, p, inverses[i]);
      if (unit.two()) e4m3_store<kVec>(to + unit.b, q, inverses[i]);
    }
  };
#pragma unroll
  for (int r = 0; r < kHeld; ++r) write(slot + r * slots, x[r], y[r], true);
  if (kCodes) __syncthreads();              // the scales are known
  if (page.to >= 0) {
#pragma unroll
    for (int r = 0; r < kHeld; ++r) write(slot + r * slots, x[r], y[r], false);
  }
  for (int i = slot + kHeld * slots; i < all; i += slots) {
    Piece u, v;
    fetch(i, u, v);
    if (i >= 2 * nh || page.to >= 0) write(i, u, v, i >= 2 * nh);
  }
  // kept rows that were not fetched ahead, now that nothing else is held
  if (kCodes && page.to >= 0)
    for (int task = warp; task < 2 * nh; task += kThreads / 32)
      if (ratios[task] != -1.f)
        append_move(reinterpret_cast<const uint8_t*>(cache_of(task, page.from)),
                    reinterpret_cast<uint8_t*>(cache_of(task, page.to)), a.c_st, page.kept, a.width,
                    a.code_bytes, ratios[task]);
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
  a.code_bytes = a.width % 16 == 0 && cache == 16 ? 16 : a.width % 8 == 0 && cache >= 8 ? 8 : 1;
  if (a.offsets) {
    // a key and a value head for each pair of warps, up to four times as many while that
    // leaves CTAs for every SM (two prompts of 42 tokens, 21/3 heads of 64: 11.3 -> 7 us)
    const int most = (a.kv_heads + 1) / 2;   // groups
    const int wanted = (int)std::max<int64_t>(4 * 148 / std::max<int64_t>(units, 1), (a.kv_heads + 7) / 8);
    const int split = std::max(1, std::min(most, wanted));
    a.heads_each = (a.kv_heads + split - 1) / split;
    a.rows = std::min({a.page, 64, 4096 / std::max(1, a.pairs)});   // a table of up to 32 KB
  } else {
    // all heads of a sequence, fewer while that leaves SMs without a CTA
    const int split = std::min(a.kv_heads, std::max(1, 2 * 148 / a.sequences));
    a.heads_each = std::min((a.kv_heads + split - 1) / split, 512);
    a.rows = 1;
  }
  const int64_t groups = ((int64_t)a.kv_heads + a.heads_each - 1) / a.heads_each;
  if (groups > 65535) return GRS_ERR_SHAPE;
  const dim3 grid((unsigned)(units + (a.clear ? 64 : 0)), (unsigned)groups);
  const int smem = (a.rows * a.pairs * 2 + (a.offsets ? 4 : 6) * a.heads_each) * (int)sizeof(float);
  return rotary_dispatch<T>(a.width, a.pairs, interleaved, alignment,
                            [&](auto vec, auto inter) -> int {
    constexpr int kVec = decltype(vec)::value;
    constexpr bool kInter = decltype(inter)::value;
    const auto kernel = a.offsets ? (codes ? append_kernel<T, kVec, kInter, true>
                                           : append_kernel<T, kVec, kInter, false>)
                                  : (codes ? append_one_kernel<T, kVec, kInter, true>
                                           : append_one_kernel<T, kVec, kInter, false>);
    kernel<<<grid, append_threads(kVec), smem, counted(stream)>>>(a);
    GRS_CUDA_CHECK_LAUNCH();
    return GRS_OK;
  });
}

}  // namespace grs

extern "C" int grs_append_tokens(
    int dtype, int cache_dtype, const void* query, int64_t q_st, int64_t q_sh, void* query_out,
    int64_t qo_st, int64_t qo_sh, int flags, const void* key, int64_t k_st, int64_t k_sh,
    const void* value, int64_t v_st, int64_t v_sh, void* key_cache, void* value_cache,
    int64_t c_sp, int64_t c_st, int64_t c_sh, float* key_scale, float* value_scale, int64_t s_sp,
    const int32_t* block_table, int64_t bt_stride, const int32_t* source_table,
    int64_t source_stride, int source_blocks, int max_blocks, const int32_t* lengths, const int32_t* offsets,
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
      source_blocks < 0 ||
      page_size <= 0 || page_size >= kMost || (int64_t)max_blocks * page_size >= kMost ||
      (!codes && source_table && (int64_t)page_size * head_width > INT_MAX) ||
      (!offsets && tokens != sequences) || (flags & GRS_APPEND_GUARDED && !status))
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
  a.source_columns = source_blocks; a.columns = max_blocks; a.lengths = lengths; a.offsets = offsets;
  a.positions = positions; a.wide = positions_are_i64;
  a.freq = frequencies; a.pairs = pairs; a.magnitude = (float)magnitude;
  // sqrt(2), rounded up: a pair's length over its larger element
  a.key_most = pairs ? (float)std::max(1.0, 1.41421366 * std::fabs(magnitude)) : 1.f;
  a.tokens = tokens; a.sequences = sequences; a.group = heads / kv_heads; a.kv_heads = kv_heads;
  a.width = head_width; a.pages = num_pages; a.page = page_size;
  a.clear = flags & GRS_APPEND_CLEAR_REST && query && offsets; a.status = status;
  a.shut = flags & GRS_APPEND_GUARDED ? status + 1 : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (sequences == 0 && !a.clear) return GRS_OK;
  return dtype == GRS_DTYPE_F32 ? append_run<float>(a, interleaved != 0, s)
                                : append_run<__nv_bfloat16>(a, interleaved != 0, s);
}
