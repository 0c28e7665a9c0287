// Grouped attention on the 5th-generation tensor cores (bf16): the prompt's
// causal rows and the slices of a shared prefix.
//
// One CTA per SM works on two "slots" of 128 rows that take turns on the
// tensor cores, so that one slot's softmax runs under the other slot's
// products.  Per 128-key block and slot: S = Q K^T (tcgen05.mma, fp32 in
// TMEM); eight softmax warps read S and write the weights back over S as bf16;
// O += P V takes the weights from TMEM.  Two threads share a row, 64 keys
// each, and exchange the row's maximum: a slot's turn is a chain of latencies
// (scores out, maximum, exponentials, weights in, products), and four softmax
// warps per scheduler hide them where two with 128 keys a thread did not.  The
// running maximum is lazy: O and the sum are rescaled only when the maximum
// has grown by more than 2^32 in weight, which fp32 sums and bf16 weights (same
// relative rounding at any exponent) do not notice.  A row's two threads exchange
// it in bf16, rounded up, and in fp32 where that rounding could reach 2^16 in
// weight (scores of 1e5: 159 instead of 94 us for 2 x 2048 tokens).  The commit that hands a
// slot its next scores also covers the slot's previous P V, so the softmax
// warps may rescale O in place without a further barrier.
//
//   warps 0-7   softmax and epilogue of slot 0      warp 16  TMA loads
//   warps 8-15  softmax and epilogue of slot 1      warps 17, 19  MMA issue
//   warp 18     zeroes the value rows behind a causal tile's last key
// The launch's 640 x 96 registers are split 104 to a softmax thread and 64 to
// the other warpgroup (512 x 104 + 128 x 64 = 61440 = 640 x 96).
// Short prompts take CTAs of one slot, two to an SM (384 x 80 registers, split 104
// to a softmax thread and 32 to the others): most of a short tile's time is its start and end,
// which then run under the other CTA's blocks.  At those 80 registers a thread
// spills 92 to 140 bytes.
//
// Causal and wide-batch slices give the slots neighbouring row tiles over one
// K/V stream (each K/V block is loaded once for 256 rows); a batch of at most
// one row tile gives both slots the same rows and halves of the slice's keys.
// Weights are rounded to bf16 for the value product; sums, statistics and
// outputs are fp32 until the one rounding of the output.
//
// 16384 tokens of 32/8 heads of 128 take 1.65 to 1.68 ms by the card, up to 1336
// TFLOP/s or 0.80 of the measured burst of the library's product; 2 x 8192 tokens 0.92 ms, of width 64
// 0.77 ms (719 TFLOP/s: half the products' work per exponential).  On 2 x 8192
// tokens the tensor pipe is active 64 % and the special-function pipe 65 % of
// the time: what remains is the chain of a slot's turn.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>
#include <mutex>

#include "grouped_attention_tc.cuh"
#include "sm100.cuh"

namespace grs {

constexpr int GTC_KEYS = 128;
constexpr int GTC_WINDOW = 260;             // offsets held for a tile's rows
constexpr float GTC_ABOVE = 16.f;           // the reference above the maximum, log2 weight

template <int DP, int kSlots>
struct GtcShape {
  static constexpr int kRow = DP >= 64 ? 128 : 64;      // bytes of a staged row
  static constexpr int kBoxes = DP * 2 / kRow;          // TMA boxes side by side
  static constexpr int kBox = 128 * kRow;
  static constexpr int kTile = kBoxes * kBox;           // Q tile, K or V block
  static constexpr int kStages = kSlots == 2 ? (DP == 128 ? 5 : DP == 64 ? 6 : 13)
                                             : (DP == 128 ? 2 : DP == 64 ? 5 : 10);
  static constexpr int kTiles = (kSlots + kStages) * kTile;
  // two slots: above half an SM's shared memory, as their 512 TMEM columns are
  // all there are; one slot: two CTAs per SM
  static_assert(kSlots == 2 ? kTiles > 114 * 1024 && kTiles <= 224 * 1024 : kTiles <= 96 * 1024,
                "CTAs per SM");
  // whether the partial sums of 16 warps pass through one Q tile
  static constexpr bool kStageFree = kTile >= 16 * 2048;
  static constexpr int kSoft = 256 * kSlots;            // softmax threads
  static constexpr int kThreads = kSoft + 128;
  static constexpr int kColumns = 256 * kSlots;         // TMEM
  static constexpr int kO = 128 * kSlots;               // first column of the outputs
};

constexpr int GTC_CAUSAL = 0, GTC_PAIR = 1, GTC_SPLIT = 2, GTC_SINGLE = 3;
constexpr int gtc_slots(int mode) { return mode == GTC_SINGLE ? 1 : 2; }

__device__ __forceinline__ float gtc_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float gtc_max3(float x, float y, float z) {
  float m;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(m) : "f"(x), "f"(y), "f"(z));
  return m;
}
__device__ __forceinline__ uint32_t gtc_pack(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// mbar_wait with its polling loop out of line: the kernel waits in many places
// and its code should stay near the size of the instruction caches (the first
// form, with everything unrolled in line, ran its once-per-tile parts at a
// quarter of their issue rate)
__device__ __noinline__ bool gtc_wait_more(uint64_t* bar, uint32_t parity) {
  return sm100::mbar_wait(bar, parity);
}
__device__ __forceinline__ bool gtc_wait(uint64_t* bar, uint32_t parity) {
  return sm100::mbar_try_wait(bar, parity) || gtc_wait_more(bar, parity);
}

// How many of the ascending offsets are <= p, by one warp
__device__ __forceinline__ int offsets_up_to(const int32_t* __restrict__ offsets, int count,
                                             int p) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = count;
  while (hi - lo > 32) {
    const int step = (hi - lo + 31) / 32;
    const int64_t at = lo + (int64_t)lane * step;
    const int n = __popc(__ballot_sync(0xffffffffu, at < hi && __ldg(offsets + at) <= p));
    if (n == 0) return lo;
    hi = (int)min((int64_t)hi, lo + (int64_t)n * step);
    lo += (n - 1) * step + 1;
  }
  const bool in = lo + lane < hi && __ldg(offsets + lo + lane) <= p;
  return lo + __popc(__ballot_sync(0xffffffffu, in));
}

// The two warps of 32 rows exchange the rows' maxima in fp32, over their bf16
// ones in shared memory: they meet before and behind it, three phases of `pair`
// from phase `met` on.  Returns the larger maximum.  A wait that gives up sets
// `failed`, which ends the stream of blocks.  Out of line like gtc_wait_more: in
// line, prompts took 1.5 to 2 % longer.
__device__ __noinline__ float gtc_exact_top(float mine, float* maxima, int half, uint64_t* pair,
                                            int met, int* failed) {
  bool ok = true;
  const auto meet = [&](int phase) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) sm100::mbar_arrive(pair);
    if (ok) ok = sm100::mbar_wait_warp(pair, phase & 1);
  };
  meet(met);
  if (ok) maxima[half * 32] = mine;
  meet(met + 1);
  const float top = fmaxf(mine, maxima[(half ^ 1) * 32]);
  meet(met + 2);
  if (!ok) *failed = 1;
  return top;
}

template <int DP, int MODE>
__global__ void __launch_bounds__(GtcShape<DP, gtc_slots(MODE)>::kThreads, 3 - gtc_slots(MODE))
grouped_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ GroupedArgs<__nv_bfloat16> a, int pps) {
  using namespace sm100;
  constexpr int kSlots = gtc_slots(MODE);
  using S = GtcShape<DP, kSlots>;
  constexpr bool kCausal = MODE == GTC_CAUSAL || MODE == GTC_SINGLE, kSplit = MODE == GTC_SPLIT;
  constexpr int kAux = S::kSoft / 32;      // first warp that is not softmax
  extern __shared__ uint8_t gtc_smem_raw[];
  __shared__ __align__(8) uint64_t q_full, kv_full[S::kStages], kv_empty[S::kStages];
  __shared__ __align__(8) uint64_t s_full[2][2], p_full[2][2], drain_bar;
  __shared__ __align__(8) uint64_t turn[2];                 // slot s has issued a block
  __shared__ __align__(8) uint64_t pair_bar[8];             // the two warps of 32 rows
  __shared__ __align__(8) uint64_t last_full, last_clean;   // the causal tile's last V block
  __shared__ uint32_t tmem_slot;
  __shared__ int failed, drain_failed;
  // per softmax warp: first and last key of any row, last first and first last key
  __shared__ int4 spans[16];
  // the window of offsets; then per slot and 32 rows, which two warps share, the
  // maxima [parity][half][row] in bf16, or maxima or sums [half][row] in fp32
  __shared__ int scratch[GTC_WINDOW > 256 * kSlots ? GTC_WINDOW : 256 * kSlots];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(gtc_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ring = smem + kSlots * S::kTile;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // late causal tiles see the most keys: they start first
  int tile, h, slice;
  if (kCausal) {
    tile = gridDim.x / a.kv_heads - 1 - (int)(blockIdx.x / a.kv_heads);
    h = blockIdx.x % a.kv_heads;
    slice = 0;
  } else {
    tile = blockIdx.x;
    h = blockIdx.y;
    slice = blockIdx.z;
  }
  const int p_tile = tile * (kSplit ? pps : kSlots * pps);    // first position
  // r / group for r < 128: exact for groups below 512
  const int per_group = (65536 + a.group - 1) / a.group;

  if (tid == S::kSoft) {
    mbar_init(&q_full, 1);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], kSplit ? 1 : kSlots);
    }
    for (int s = 0; s < 2; ++s) {
      for (int half = 0; half < 2; ++half) {
        mbar_init(&s_full[s][half], 1);
        mbar_init(&p_full[s][half], 4);
      }
    }
    mbar_init(&drain_bar, kSlots);
    for (int s = 0; s < 8; ++s) mbar_init(&pair_bar[s], 2);
    mbar_init(&turn[0], 1);
    mbar_init(&turn[1], 1);
    mbar_init(&last_full, 1);
    mbar_init(&last_clean, 1);
    failed = drain_failed = 0;
    mbar_init_fence();
    // the queries need no key range: their loads go out at once
    const int q_slots = kSplit ? 1 : kSlots;
    mbar_arrive_expect_tx(&q_full, q_slots * S::kBoxes * pps * a.group * S::kRow);
    for (int s = 0; s < q_slots; ++s)
      for (int b = 0; b < S::kBoxes; ++b)
        tma_load_3d(smem + s * S::kTile + b * S::kBox, &tm_q, b * 64, h * a.group,
                    p_tile + s * pps, &q_full);
  }
  // So does the first K block of a causal tile whose first position lies in a
  // sequence: it begins with that sequence, whatever the other rows see.
  bool k_sent = false;
  if (kCausal && warp == kAux) {
    const int n = offsets_up_to(a.offsets, a.sequences + 1, p_tile);
    k_sent = n > 0 && n <= a.sequences;
    if (k_sent && lane == 0) {
      const int key = min(max(__ldg(a.offsets + n - 1), 0), p_tile);
      mbar_arrive_expect_tx(&kv_full[0], S::kTile);
      for (int b = 0; b < S::kBoxes; ++b)
        tma_load_3d(ring + b * S::kBox, &tm_k, b * 64, h, key, &kv_full[0]);
    }
    __syncwarp();
  }
  // the kernel that joins the slices may start as SMs fall free
  if (!kCausal) asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if (warp == kAux + 1) tmem_alloc(&tmem_slot, S::kColumns);
  // The offsets that can begin or end a sequence of this tile: all of them, or
  // a window from the sequence of the first position on (found by a search of
  // one round of loads per factor of 32, where a binary search per row would
  // wait for one load per factor of 2).
  int window_at = 0, window_n = 0;
  if (kCausal && warp < kAux) {
    const int count = a.sequences + 1;
    if (count > GTC_WINDOW)
      window_at = max(0, offsets_up_to(a.offsets, count, p_tile) - 1);
    window_n = min(GTC_WINDOW, count - window_at);
    for (int i = tid; i < window_n; i += S::kSoft) scratch[i] = __ldg(a.offsets + window_at + i);
  }
  __syncthreads();
  int begin = 0, end = 0, position = -1;
  if (tid < S::kSoft) {
    const int slot = tid >> 8, r = tid & 127;
    const int p = p_tile + (kSplit ? 0 : slot * pps) + ((r * per_group) >> 16);
    if (r < pps * a.group && p < a.positions) position = p;
    if (kCausal) {
      if (position >= 0) {
        int from = 0, to = window_n;       // first window entry past p
        while (from < to) {
          const int mid = (from + to) >> 1;
          if (scratch[mid] <= position) from = mid + 1; else to = mid;
        }
        if (from == window_n && window_at + window_n <= a.sequences) {
          // sequences without tokens filled the window
          causal_range(a.offsets, a.sequences, position, begin, end);
        } else if (from > 0 && from < window_n) {
          begin = min(max(scratch[from - 1], 0), position);
          end = position + 1;
        }
      }
    } else {
      begin = slice * a.slice_keys;
      end = max(begin, min(a.keys, begin + a.slice_keys));
      if (kSplit) {
        const int blocks = (end - begin + GTC_KEYS - 1) / GTC_KEYS;
        const int mid = min(end, begin + (blocks + 1) / 2 * GTC_KEYS);
        if (slot == 0) end = mid; else begin = mid;
      }
      if (!kSplit && p_tile + slot * pps >= a.positions) end = begin;
    }
    const bool any = end > begin;
    const int4 span = make_int4(__reduce_min_sync(0xffffffffu, any ? begin : INT_MAX),
                                __reduce_max_sync(0xffffffffu, any ? end : 0),
                                __reduce_max_sync(0xffffffffu, any ? begin : 0),
                                __reduce_min_sync(0xffffffffu, any ? end : INT_MAX));
    if (lane == 0) spans[warp] = span;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  int lo_key[2], hi_key[2], in_lo[2], in_hi[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (s >= kSlots) {
      lo_key[s] = in_hi[s] = INT_MAX;
      hi_key[s] = in_lo[s] = 0;
      continue;
    }
    const int4 w0 = spans[8 * s], w1 = spans[8 * s + 1], w2 = spans[8 * s + 2],
               w3 = spans[8 * s + 3];
    lo_key[s] = min(min(w0.x, w1.x), min(w2.x, w3.x));
    hi_key[s] = max(max(w0.y, w1.y), max(w2.y, w3.y));
    in_lo[s] = max(max(w0.z, w1.z), max(w2.z, w3.z));
    in_hi[s] = min(min(w0.w, w1.w), min(w2.w, w3.w));
  }
  // block ranges [first[s], last[s]) of 128 keys from origin[s]
  int origin[2], first[2], last[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const bool any = hi_key[s] > lo_key[s];
    origin[s] = kSplit ? (any ? lo_key[s] : 0) : min(lo_key[0], lo_key[1]);
    first[s] = any ? (lo_key[s] - origin[s]) / GTC_KEYS : 0;
    last[s] = any ? (hi_key[s] - origin[s] + GTC_KEYS - 1) / GTC_KEYS : 0;
  }
  // the K/V stream of a pair covers both slots' blocks
  const bool any0 = last[0] > first[0], any1 = last[1] > first[1];
  const int lo = any0 && any1 ? min(first[0], first[1]) : any0 ? first[0] : first[1];
  const int hi = any0 && any1 ? max(last[0], last[1]) : any0 ? last[0] : last[1];
  // Value rows past the tile's last key (rows behind the last sequence, the
  // next sequence, later tokens) meet only zero weights, but they may hold
  // NaN: the last V block is cleared of them before its product.
  const int end_row = kCausal && (any0 || any1)
                          ? max(hi_key[0], hi_key[1]) - origin[0] - (hi - 1) * GTC_KEYS
                          : GTC_KEYS;
  const bool clear = end_row % 16 != 0;
  volatile int* gave_up = &failed;

  if (warp >= kAux) {
    if (kSlots == 2)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n");
    else
      asm volatile("setmaxnreg.dec.sync.aligned.u32 32;\n");
    if (warp == kAux) {
      if (lane == 0) {                   // TMA producer
        // order of the ring: per block and stream V(j), K(j + 1)
        int g = k_sent ? 1 : 0;
        unsigned armed = k_sent ? 1 : 0; // stages with a load, their last phase in `phase`
        unsigned phase = 0;
        bool last_armed = false;
#pragma unroll 1
        for (int n = 0; n < 2 * (kSplit ? 2 : 1) * (hi - lo + 1); ++n) {
          // pair: (block, K or V); split: (block, slot, K or V)
          const int s = kSplit ? (n >> 1) & 1 : 0, is_k = n & 1;
          const int j = lo - 1 + (kSplit ? n >> 2 : n >> 1) + is_k;
          const int end_j = kSplit ? (s ? last[1] : last[0]) : hi;
          if (j < lo || j >= end_j || (k_sent && j == lo && is_k)) continue;
          const int st = g % S::kStages, r = g / S::kStages;
          if (*gave_up) break;
          if (r > 0 && !gtc_wait(&kv_empty[st], (r - 1) & 1)) {
            failed = 1;
            break;
          }
          const bool is_last = kCausal && clear && !is_k && j == hi - 1;
          uint64_t* bar = is_last ? &last_full : &kv_full[st];
          mbar_arrive_expect_tx(bar, S::kTile);
          const int key = (kSplit && s ? origin[1] : origin[0]) + j * GTC_KEYS;
#pragma unroll
          for (int b = 0; b < S::kBoxes; ++b)
            tma_load_3d(ring + st * S::kTile + b * S::kBox, is_k ? &tm_k : &tm_v, b * 64, h, key,
                        bar);
          if (is_last) {
            last_armed = true;
          } else {
            armed |= 1u << st;
            phase = (phase & ~(1u << st)) | (unsigned)(r & 1) << st;
          }
          ++g;
        }
        // every load in flight lands before the CTA exits
        if (!gtc_wait(&q_full, 0)) drain_failed = 1;
        if (last_armed && !gtc_wait(&last_full, 0)) drain_failed = 1;
#pragma unroll 1
        for (int s = 0; s < S::kStages; ++s)
          if (((armed >> s) & 1) && !gtc_wait(&kv_full[s], (phase >> s) & 1)) drain_failed = 1;
      }
    } else if (warp == kAux + 1 || (kSlots == 2 && warp == kAux + 3)) {   // MMA issuer of a slot
      // A warp per slot: what it computes between two blocks runs under the
      // other slot's products.  The two issue in turn, which keeps the slots half
      // a period apart (without the turns they fall into step, both in their
      // softmax, then both waiting for products: 1.87 against 1.73 ms on 16384
      // tokens).  The whole warp walks the loop and one elected lane issues, so
      // that addresses and descriptors can stay in uniform registers.  Per block
      // the slot issues P V of its first 64 keys and the next scores for 64 keys,
      // then the same for the other 64: each half of the softmax warps waits for
      // its own half only.
      const int s = warp == kAux + 1 ? 0 : 1;
      uint32_t elected;
      asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n"
                   : "=r"(elected));
      const bool lead = elected != 0;
      constexpr uint32_t i_pv = idesc_bf16_f32(128, DP) | IDESC_B_MN;
      constexpr int kPerBox = S::kRow / 32;             // 16-element steps of a box
      const int first_s = s ? first[1] : first[0], last_s = s ? last[1] : last[0];
      // products of the slot's last block stop at its last key, in steps of 16
      const int tail = ((s ? hi_key[1] : hi_key[0]) - (s ? origin[1] : origin[0]) -
                        (last_s - 1) * GTC_KEYS + 15) / 16;
      const uint64_t q_desc = smem_desc(smem + (kSplit ? 0 : s) * S::kTile, S::kRow, 16,
                                        8 * S::kRow);
      const uint64_t k_desc = smem_desc(ring, S::kRow, 16, 8 * S::kRow);
      const uint64_t v_desc = smem_desc(ring, S::kRow, S::kBox, 8 * S::kRow);
      const uint32_t t_s = tmem + s * GTC_KEYS, t_o = tmem + S::kO + s * DP;
      int next = 0;                                     // ring stage and phase bit
      uint32_t ph = 0;
      bool ok = any0 || any1;
      if (ok) ok = mbar_wait(&q_full, 0);
      const auto advance = [&] {
        if (++next == S::kStages) next = 0, ph ^= 1;
      };
      // the other slot of a split fetches its own blocks in between
      const int last_o = s ? last[0] : last[1];
      const auto skip = [&](int j) {
        if (j >= 0 && j < last_o) advance();
        if (j + 1 < last_o) advance();
      };
#pragma unroll 1
      for (int j = lo - 1; j < hi && ok; ++j) {         // P V of block j, Q K of block j + 1
        const bool v_mine = j >= first_s && j < last_s;
        const bool k_mine = j + 1 >= first_s && j + 1 < last_s;
        const bool v_here = kSplit ? v_mine : j >= lo;
        const bool k_here = kSplit ? k_mine : j + 1 < hi;
        if (kSplit && s == 1) skip(j);
        int v_st = 0, k_st = 0;
        if (v_here) {
          v_st = next;
          ok = kCausal && clear && j == hi - 1 ? mbar_wait(&last_clean, 0)
                                               : mbar_wait(&kv_full[v_st], ph);
          advance();
        }
        if (k_here) {
          k_st = next;
          if (ok) ok = mbar_wait(&kv_full[k_st], ph);
          advance();
        }
        if (kSplit && s == 0) skip(j);
        const int i = j - first_s;
        const bool v_last = j == last_s - 1, k_last = j + 2 == last_s;
        const uint64_t vd = v_desc + v_st * (S::kTile >> 4);
        const uint64_t kd = k_desc + k_st * (S::kTile >> 4);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (ok && v_mine) ok = mbar_wait(&p_full[s][half], i & 1);
          if (kSlots == 2 && ok && half == 0) {   // this slot's turn of block j
            const int turns = j - lo + 1;
            if (s == 1)
              ok = mbar_wait(&turn[0], turns & 1);
            else if (turns > 0)
              ok = mbar_wait(&turn[1], (turns - 1) & 1);
          }
          if (!ok) break;
          tc_fence_after();
          if (lead) {
            if (v_mine) {
              const uint64_t vh = vd + half * ((64 * S::kRow) >> 4);
              const uint32_t t_p = t_s + 64 * half;
              if (!v_last) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                  mma_bf16_tmem_a(t_o, t_p + kk * 8, vh + kk * ((16 * S::kRow) >> 4), i_pv,
                                  i > 0 || half > 0 || kk > 0);
              } else {
#pragma unroll 1
                for (int kk = 0; kk < min(tail - 4 * half, 4); ++kk)
                  mma_bf16_tmem_a(t_o, t_p + kk * 8, vh + kk * ((16 * S::kRow) >> 4), i_pv,
                                  i > 0 || half > 0 || kk > 0);
                if (half == 1) {
                  mma_commit(&s_full[s][0]);
                  mma_commit(&s_full[s][1]);
                }
              }
            }
            if (k_mine) {
              const uint64_t kh = kd + half * ((64 * S::kRow) >> 4);
              const uint32_t i_qk =
                  idesc_bf16_f32(128, k_last ? max(1, min(tail - 4 * half, 4)) * 16 : 64);
#pragma unroll
              for (int kk = 0; kk < DP / 16; ++kk) {
                const uint32_t off = ((kk / kPerBox) * S::kBox + (kk % kPerBox) * 32) >> 4;
                mma_bf16(t_s + 64 * half, q_desc + off, kh + off, i_qk, kk > 0);
              }
              mma_commit(&s_full[s][half]);
            }
          }
        }
        if (!ok) break;
        if (lead) {
          mbar_arrive(&turn[s]);
          // a stage is free when both slots of a pair are done with it
          if (v_mine) mma_commit(&kv_empty[v_st]); else if (v_here) mbar_arrive(&kv_empty[v_st]);
          if (k_mine) mma_commit(&kv_empty[k_st]); else if (k_here) mbar_arrive(&kv_empty[k_st]);
        }
      }
      if (!ok && (any0 || any1)) failed = 1;
      // no MMA may still use TMEM or shared memory when they are given back
      if (lead) mma_commit(&drain_bar);
      if (!mbar_wait(&drain_bar, 0)) drain_failed = 1;
    } else if (kCausal && warp == kAux + 2 && clear) {
      const int at = 1 + 2 * (hi - 1 - lo);   // its place in the ring
      // (the stream may still be a whole tile's work away from its last block; the
      // lanes may read the flag at different times, the warp leaves as one)
      bool ok = false;
      while (!ok && !__any_sync(0xffffffffu, *gave_up)) ok = mbar_wait_warp(&last_full, 0);
      if (ok) {
        uint8_t* block = ring + (at % S::kStages) * S::kTile;
        constexpr int kPieces = S::kRow / 16;
        for (int b = 0; b < S::kBoxes; ++b)
          for (int i = end_row * kPieces + lane; i < (end_row + 15) / 16 * 16 * kPieces; i += 32)
            *reinterpret_cast<uint4*>(block + b * S::kBox + i * 16) = make_uint4(0, 0, 0, 0);
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&last_clean);
      }
    }
  } else {                               // softmax and epilogue, two threads per row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n");
    const int slot = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3, r = tid & 127;
    const int blocks = slot == 0 ? last[0] - first[0] : last[1] - first[1];
    const int key_first = (slot == 0 ? origin[0] + first[0] * GTC_KEYS
                                     : origin[1] + first[1] * GTC_KEYS) + 64 * half;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_s = tmem + lanes + slot * GTC_KEYS;
    const float c = a.scale_log2, slack = 32.f / c;
    const int all_from = slot == 0 ? in_lo[0] : in_lo[1];
    const int all_to = slot == 0 ? in_hi[0] : in_hi[1];
    // this thread's half of the output columns, in runs of kCols
    constexpr int kCols = DP == 32 ? 16 : 32, kRuns = DP / 2 / kCols;
    const uint32_t t_o = tmem + lanes + S::kO + slot * DP + half * (DP / 2);
    int* shared32 = scratch + slot * 256 + quarter * 64;
    __nv_bfloat16* tops = reinterpret_cast<__nv_bfloat16*>(shared32) + lane;
    float* sums = reinterpret_cast<float*>(shared32) + lane;
    uint64_t* pair = &pair_bar[slot * 4 + quarter];
    const auto tell = [&] {                // own value is in shared memory
      __syncwarp();
      if (lane == 0) mbar_arrive(pair);
    };
    const float2 c2 = make_float2(c, c);
    uint32_t raw[2][32];
    // this thread's 64 scores, masked; returns their maximum
    const auto scores = [&](int i, bool& dead) {
      tmem_load32_async(t_s + 64 * half, raw[0]);
      tmem_load32_async(t_s + 64 * half + 32, raw[1]);
      tmem_loaded32(raw[0]);
      tmem_loaded32(raw[1]);
      const int key0 = key_first + i * GTC_KEYS;
      dead = false;                        // no row of the warp sees any of its 64 keys
      if (key0 < all_from || key0 + 64 > all_to) {
        const int from = begin - key0, to = end - key0;
        dead = !__any_sync(0xffffffffu, max(from, 0) < min(to, 64));
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          // bit j: key 32 q + j is seen
          const int f = min(max(from - 32 * q, 0), 32), e = min(max(to - 32 * q, 0), 32);
          const uint32_t seen_bits =
              (e == 32 ? 0xffffffffu : (1u << e) - 1u) & (f == 32 ? 0u : 0xffffffffu << f);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (!(seen_bits & (1u << j))) raw[q][j] = 0xff800000u;
        }
      }
      float t4[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t* v = &raw[q >> 1][16 * (q & 1)];
        t4[q] = fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
#pragma unroll
        for (int j = 2; j < 16; j += 2)
          t4[q] = gtc_max3(t4[q], __uint_as_float(v[j]), __uint_as_float(v[j + 1]));
      }
      return gtc_max3(fmaxf(t4[0], t4[1]), t4[2], t4[3]);
    };
    // weights exp2(c s - base) of the scores in raw, packed into raw[0]; returns
    // their sum.  Groups of 16 scores pass through three stages (scale,
    // exponential, sum and pack) one behind the other: in the order of the
    // formula every pair waits for its own exponential.
    const auto weights = [&](float base) {
      const float2 b2 = make_float2(-base, -base);
      float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
      const auto exps = [&](int g) {
        uint32_t* v = &raw[g >> 1][16 * (g & 1)];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 x = __ffma2_rn(
              make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), c2, b2);
          v[2 * j] = __float_as_uint(x.x);
          v[2 * j + 1] = __float_as_uint(x.y);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[2 * j] = __float_as_uint(gtc_exp2(__uint_as_float(v[2 * j])));
          v[2 * j + 1] = __float_as_uint(gtc_exp2(__uint_as_float(v[2 * j + 1])));
        }
      };
      const auto pack = [&](int g) {
        uint32_t* v = &raw[g >> 1][16 * (g & 1)];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 x = make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
          if (j & 1) sum1 = __fadd2_rn(sum1, x); else sum0 = __fadd2_rn(sum0, x);
          raw[0][8 * g + j] = gtc_pack(x.x, x.y);
        }
      };
      exps(0);
#pragma unroll
      for (int g = 1; g < 4; ++g) {
        exps(g);
        pack(g - 1);
      }
      pack(3);
      sum0 = __fadd2_rn(sum0, sum1);
      return sum0.x + sum0.y;
    };
    float m = -INFINITY, l = 0.f;
    int met = 0;                           // phases of the pair's barrier
    bool ok = true;
    const auto meet = [&] {
      ok = mbar_wait_warp(pair, met & 1);
      ++met;
    };
    // Where `top`, from bf16, can lie more than 2^16 in weight above the row's
    // maximum (bf16 steps are up to 2^-7 of the value), the pair exchanges the
    // maxima themselves: rows with scores beyond 2^14 in the exponent of 2 would
    // lose every weight.  Both threads of a row know the same `top`, so both warps
    // do this or neither.
    const auto exact = [&](float& top, float mine) {
      const bool far =
          position >= 0 && top > -INFINITY && fabsf(top) * c > 128.f * GTC_ABOVE;
      if (!__any_sync(0xffffffffu, far)) return;
      top = gtc_exact_top(mine, sums, half, pair, met, &failed);
      met += 3;
    };
#pragma unroll 1
    for (int i = 0; i < blocks; ++i) {
      if (!(ok = mbar_wait_warp(&s_full[slot][half], i & 1))) break;
      tc_fence_after();
      bool dead;
      // The reference maximum need not be exact, only the same for both threads
      // of a row and near enough to the maximum: it passes between them in bf16,
      // rounded up.  (Two copies: the partner may be one block behind, not two.)
      const float mine = scores(i, dead);
      __nv_bfloat16* at = tops + (i & 1) * 64;
      at[half * 32] = __float2bfloat16_ru(mine);
      tc_fence_before();
      tell();
      // The weights are taken against the maximum so far; the partner's part of
      // this block's maximum is read behind them.  Only where the maximum has
      // grown by more than 2^32 in weight (and in a row's first block) are the
      // scores read again and the sums rescaled.
      float part = 0.f;
      const float before = m;
      if (i > 0 && !dead) part = weights(m == -INFINITY ? 0.f : m * c);
      meet();
      if (!ok) break;
      float top = fmaxf(__bfloat162float(__float2bfloat16_ru(mine)),
                        __bfloat162float(at[(half ^ 1) * 32]));
      bool grown = top > m + slack;
      if (i == 0) {
        exact(top, mine);
        m = top;
        if (!dead) part = weights(m == -INFINITY ? 0.f : m * c);
      } else if (__any_sync(0xffffffffu, grown)) {
        // Both threads of the row are here with their scores of this block, so
        // every product into O is done, and none starts before both are through.
        exact(top, mine);
        tc_fence_after();
        grown = top > m + slack;
        if (grown) m = top;
        // the difference of what the weights are taken against, as it rounded there
        const float keep = grown ? gtc_exp2(__fmul_rn(before, c) - __fmul_rn(m, c)) : 1.f;
        l *= keep;
#pragma unroll 1
        for (int q = 0; q < DP / 2; q += 16) {
          uint32_t o[16];
          tmem_load16_async(t_o + q, o);
          tmem_loaded16(o);
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
          tmem_store16(t_o + q, o);
        }
        tmem_stored();
        scores(i, dead);
        if (!dead) part = weights(m == -INFINITY ? 0.f : m * c);
        tc_fence_before();
        tell();
        meet();
        if (!ok) break;
        tc_fence_after();
      }
      if (dead) {
#pragma unroll
        for (int j = 0; j < 32; ++j) raw[0][j] = 0;
      }
      l += part;
      tmem_store32(t_s + 64 * half, raw[0]);   // over the thread's own scores
      tmem_stored();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[slot][half]);
    }
    // the slot's last products are done; without any, its queries have landed
    // (the outputs are staged over them)
    if (ok) ok = blocks > 0 ? mbar_wait_warp(&s_full[slot][half], blocks & 1)
                            : mbar_wait_warp(&q_full, 0);
    tc_fence_after();
    // both warps have stored their last weights, so the maxima are read
    sums[half * 32] = l;
    tell();
    if (ok) meet();
    if (!ok) failed = 1;
    l += sums[(half ^ 1) * 32];
    const bool seen = end > begin && position >= 0;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int head = h * a.group + r - ((r * per_group) >> 16) * a.group;
    if constexpr (kCausal) {
      // the output row goes through the slot's Q tile (its products are done)
      // so that whole rows leave in 16-byte pieces of neighbouring lanes
      constexpr int kPieces = DP / 16;     // of this half
      uint8_t* stage = smem + slot * S::kTile;
      const auto piece = [&](int row, int at) {
        const int x = DP >= 64 ? row & 7 : (row >> 1) & 3;
        return reinterpret_cast<uint4*>(stage + row * (DP * 2) + (((half * kPieces + at) ^ x) << 4));
      };
      bool odd = seen && !(fabsf(l) <= FLT_MAX);
      float2 nil = make_float2(0.f, 0.f);  // stays 0 while every output is finite
#pragma unroll 1
      for (int q = 0; q < kRuns; ++q) {
        uint32_t o[kCols];
        if (blocks > 0) {
          if constexpr (kCols == 32) {
            tmem_load32_async(t_o + 32 * q, o);
            tmem_loaded32(o);
          } else {
            tmem_load16_async(t_o, o);
            tmem_loaded16(o);
          }
        }
#pragma unroll
        for (int k = 0; k < kCols / 8; ++k) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float2 x = __fmul2_rn(make_float2(__uint_as_float(o[8 * k + 2 * j]),
                                              __uint_as_float(o[8 * k + 2 * j + 1])),
                                  make_float2(inv, inv));
            nil = __ffma2_rn(x, make_float2(0.f, 0.f), nil);
            w[j] = seen ? gtc_pack(x.x, x.y) : 0u;
          }
          *piece(r, kCols / 8 * q + k) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      odd |= seen && !(nil.x + nil.y == 0.f);
      __syncwarp();
      const bool mine = position >= 0 && (seen || a.clear_rest);
      const unsigned write = __ballot_sync(0xffffffffu, mine && ok);
      unsigned again = __ballot_sync(0xffffffffu, odd && seen && ok);
      const int64_t to = (int64_t)position * a.o_sp + (int64_t)head * a.o_sh;
      const int at = lane % kPieces, column = half * (DP / 2) + at * 8;
#pragma unroll 4
      for (int i = 0; i < 32; i += 32 / kPieces) {
        const int rr = i + lane / kPieces;
        const int64_t off = __shfl_sync(0xffffffffu, to, rr);
        if (((write >> rr) & 1) && column < a.D)
          *reinterpret_cast<uint4*>(a.out + off + column) = *piece(quarter * 32 + rr, at);
      }
      __syncwarp();
      while (again) {
        const int rr = __ffs(again) - 1;
        again &= again - 1;
        causal_row_again<__nv_bfloat16, (DP + 63) / 64>(
            a, __shfl_sync(0xffffffffu, position, rr), __shfl_sync(0xffffffffu, head, rr),
            __shfl_sync(0xffffffffu, begin, rr), __shfl_sync(0xffffffffu, end, rr),
            half * (DP / 2), min(a.D, (half + 1) * (DP / 2)));
      }
    } else {
      // 16 columns of the warp's 32 rows at a time pass through 2 KB of shared
      // memory: written from the rows' own threads, a warp's store would touch
      // 32 rows with 16 bytes each, and 6.6 of 15 us of a three-block slice went
      // into that.  The Q tile is free in a pair (the slot's scores are done); a
      // split leaves the second one unused.
      const int part = kSplit ? 2 * slice + slot : slice;
      const int64_t at = ((int64_t)part * a.positions + position) * a.heads + head;
      uint8_t* stage = S::kStageFree ? smem + (kSplit ? S::kTile + warp * 2048
                                                      : slot * S::kTile + (warp & 7) * 2048)
                                     : ring + S::kStages * S::kTile + warp * 2048;
      const unsigned write = __ballot_sync(0xffffffffu, position >= 0 && ok);
#pragma unroll 1
      for (int q = 0; q < DP / 2; q += 16) {
        uint32_t o[16];
        if (blocks > 0) {
          tmem_load16_async(t_o + q, o);
          tmem_loaded16(o);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (blocks > 0)
            x = make_float4(__uint_as_float(o[4 * j]) * inv, __uint_as_float(o[4 * j + 1]) * inv,
                            __uint_as_float(o[4 * j + 2]) * inv,
                            __uint_as_float(o[4 * j + 3]) * inv);
          *reinterpret_cast<float4*>(stage + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = x;
        }
        __syncwarp();
        const int column = half * (DP / 2) + q + 4 * (lane & 3);
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          const int rr = i + (lane >> 2);
          const int64_t to = __shfl_sync(0xffffffffu, at, rr) * a.D + column;
          if (((write >> rr) & 1) && column < a.D)
            *reinterpret_cast<float4*>(a.part + to) = *reinterpret_cast<const float4*>(
                stage + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
        }
        __syncwarp();
      }
      if (position >= 0 && ok && half == 0)
        a.part_lse[at] = l == 0.f ? -INFINITY : __fmul_rn(m, c) + log2f(l);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kAux + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kColumns);
  }
  if (tid == 0 && (failed || drain_failed)) set_status(a.status, GRS_ERR_TIMEOUT);
}

// ---- host --------------------------------------------------------------------
namespace {

PFN_cuTensorMapEncodeTiled_v12000 gtc_encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// [rows, heads, D] with row and head strides in elements, in boxes of
// box_cols x box_heads x box_rows; a dimension of one row keeps no stride
bool gtc_map(CUtensorMap* map, const void* base, int64_t rows, int64_t heads, int D, int64_t st,
             int64_t sh, int box_cols, int box_heads, int box_rows) {
  auto fn = gtc_encode();
  if (!fn) return false;
  const int64_t one = (D + 7) / 8 * 8;
  if (heads == 1) sh = one;
  if (rows == 1) st = one;
  cuuint64_t dim[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t str[2] = {(cuuint64_t)sh * 2, (cuuint64_t)st * 2};
  cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
  cuuint32_t est[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dim, str, box, est,
            CU_TENSOR_MAP_INTERLEAVE_NONE,
            box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// rows that TMA can fetch: 16-byte aligned, positive strides of whole 16 bytes
bool gtc_rows_ok(const void* base, int64_t rows, int64_t st, int64_t heads, int64_t sh, int D) {
  const auto ok = [](int64_t n, int64_t s) {
    return n == 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38));
  };
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && D % 8 == 0 && ok(rows, st) &&
         ok(heads, sh);
}

template <int DP, int MODE>
int gtc_launch(const GroupedArgs<__nv_bfloat16>& args, cudaStream_t stream) {
  constexpr int kSlots = gtc_slots(MODE);
  using S = GtcShape<DP, kSlots>;
  GroupedArgs<__nv_bfloat16> a = args;
  const int pps = 128 / a.group;                        // positions of a slot
  const int cols = S::kRow / 2;
  // a zero scale weighs every key alike; masked scores must stay -inf
  a.scale_log2 = std::max(a.scale_log2, 1e-30f);
  CUtensorMap q, k, v;
  if (!gtc_map(&q, a.q, a.positions, a.heads, a.D, a.q_sp, a.q_sh, cols, a.group, pps) ||
      !gtc_map(&k, a.k, a.keys, a.kv_heads, a.D, a.k_st, a.k_sh, cols, 1, GTC_KEYS) ||
      !gtc_map(&v, a.v, a.keys, a.kv_heads, a.D, a.v_st, a.v_sh, cols, 1, GTC_KEYS))
    return GRS_ERR_SHAPE;
  constexpr bool kCausal = MODE == GTC_CAUSAL || MODE == GTC_SINGLE;
  const int step = pps * (MODE == GTC_SPLIT ? 1 : kSlots);
  const int64_t tiles = ((int64_t)a.positions + step - 1) / step;
  if (tiles * a.kv_heads > INT_MAX || (!kCausal && (a.kv_heads > 65535 || a.slices > 65535)))
    return GRS_ERR_SHAPE;
  const dim3 grid = kCausal ? dim3((unsigned)(tiles * a.kv_heads))
                            : dim3((unsigned)tiles, a.kv_heads, a.slices);
  // the tiles start at the first 1024-byte boundary behind the static variables
  static std::atomic<int> smem_of[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return GRS_ERR_CUDA;
  int smem = smem_of[dev].load(std::memory_order_acquire);
  if (smem == 0) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, grouped_tc_kernel<DP, MODE>) != cudaSuccess)
      return GRS_ERR_CUDA;
    const int fixed = (int)fa.sharedSizeBytes;
    smem = (fixed + 1023) / 1024 * 1024 - fixed + S::kTiles +
           (!kCausal && !S::kStageFree ? 16 * 2048 : 0);
    if (cudaFuncSetAttribute(grouped_tc_kernel<DP, MODE>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return GRS_ERR_CUDA;
    smem_of[dev].store(smem, std::memory_order_release);
  }
  grouped_tc_kernel<DP, MODE><<<grid, S::kThreads, smem, counted(stream)>>>(q, k, v, a, pps);
  GRS_CUDA_CHECK_LAUNCH();
  return GRS_OK;
}

template <int MODE>
int gtc_width(const GroupedArgs<__nv_bfloat16>& a, cudaStream_t stream) {
  if (a.D <= 32) return gtc_launch<32, MODE>(a, stream);
  if (a.D <= 64) return gtc_launch<64, MODE>(a, stream);
  return gtc_launch<128, MODE>(a, stream);
}

}  // namespace

bool grouped_tc_takes(const GroupedArgs<__nv_bfloat16>& a) {
  return a.D <= 128 && a.group <= 128 && a.scale_log2 >= 0.f &&
         gtc_rows_ok(a.q, a.positions, a.q_sp, a.heads, a.q_sh, a.D) &&
         gtc_rows_ok(a.k, a.keys, a.k_st, a.kv_heads, a.k_sh, a.D) &&
         gtc_rows_ok(a.v, a.keys, a.v_st, a.kv_heads, a.v_sh, a.D) &&
         (a.offsets == nullptr || gtc_rows_ok(a.out, a.positions, a.o_sp, a.heads, a.o_sh, a.D));
}

int grouped_tc_launch(const GroupedArgs<__nv_bfloat16>& a, cudaStream_t stream) {
  if (a.offsets) {
    // One slot per CTA where pairs would leave SMs without work (one prompt of
    // 512 tokens, 32/8 heads: 18.8 -> 13.3 us) or hold mostly different
    // sequences (500 prompts of up to 64: 60 -> 55 us); pairs read K and V half as
    // often (8 x 1024 tokens: 106 against 119 us).
    const int pps = 128 / a.group;
    const int64_t pairs = ((int64_t)a.positions + 2 * pps - 1) / (2 * pps) * a.kv_heads;
    return pairs < 148 || (int64_t)a.positions < 128ll * a.sequences
               ? gtc_width<GTC_SINGLE>(a, stream) : gtc_width<GTC_CAUSAL>(a, stream);
  }
  return grouped_tc_split(a.positions, a.group) ? gtc_width<GTC_SPLIT>(a, stream)
                                                : gtc_width<GTC_PAIR>(a, stream);
}

}  // namespace grs
