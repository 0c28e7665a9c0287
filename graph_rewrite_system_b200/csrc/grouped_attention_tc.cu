// Grouped attention on the 5th-generation tensor cores (bf16): the prompt's
// causal rows and the slices of a shared prefix.
//
// One CTA per SM works on two "slots" of 128 rows that take turns on the
// tensor cores, so that one slot's softmax runs under the other slot's
// products.  Per 128-key block and slot: S = Q K^T (tcgen05.mma, fp32 in
// TMEM); four softmax warps read S, one row per thread, and write the weights
// back over S as bf16; O += P V takes the weights from TMEM.  The running
// maximum is lazy: O and the sum are rescaled only when the maximum has grown
// by more than 2^8 in weight, which fp32 sums and bf16 weights (same relative
// rounding at any exponent) do not notice.  The commit that hands a slot its
// next scores also covers the slot's previous P V, so the softmax warps may
// rescale O in place without a further barrier.
//
//   warps 0-3   softmax and epilogue of slot 0      warp 8  TMA loads
//   warps 4-7   softmax and epilogue of slot 1      warp 9  MMA issue
//   warp 10     zeroes the value rows behind a causal tile's last key
// The launch's 384 x 168 registers are split 216 to a softmax thread, which
// holds a row's 128 scores, and 72 to the other warpgroup (256 x 216 + 128 x
// 72 = 64512 = 384 x 168).
//
// Causal and wide-batch slices give the slots neighbouring row tiles over one
// K/V stream (each K/V block is loaded once for 256 rows); a batch of at most
// one row tile gives both slots the same rows and halves of the slice's keys.
// Weights are rounded to bf16 for the value product; sums, statistics and
// outputs are fp32 until the one rounding of the output.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <mutex>

#include "grouped_attention_tc.cuh"
#include "sm100.cuh"

namespace grs {

constexpr int GTC_THREADS = 384, GTC_KEYS = 128;
constexpr int GTC_O = 256;                  // first TMEM column of the outputs

template <int DP>
struct GtcShape {
  static constexpr int kRow = DP >= 64 ? 128 : 64;      // bytes of a staged row
  static constexpr int kBoxes = DP * 2 / kRow;          // TMA boxes side by side
  static constexpr int kBox = 128 * kRow;
  static constexpr int kTile = kBoxes * kBox;           // Q tile, K or V block
  static constexpr int kStages = DP == 128 ? 5 : DP == 64 ? 6 : 13;
  // above half an SM's shared memory: the 512 TMEM columns are one CTA's
  static constexpr int kSmem = (2 + kStages) * kTile + 1024;
  static_assert(kSmem > 116 * 1024 && kSmem <= 227 * 1024, "one CTA per SM");
};

constexpr int GTC_CAUSAL = 0, GTC_PAIR = 1, GTC_SPLIT = 2;

__device__ __forceinline__ float gtc_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t gtc_pack(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <int DP, int MODE>
__global__ void __launch_bounds__(GTC_THREADS, 1)
grouped_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, GroupedArgs<__nv_bfloat16> a, int pps,
                  int negate) {
  using namespace sm100;
  using S = GtcShape<DP>;
  constexpr bool kCausal = MODE == GTC_CAUSAL, kSplit = MODE == GTC_SPLIT;
  extern __shared__ uint8_t gtc_smem_raw[];
  __shared__ __align__(8) uint64_t q_full, kv_full[S::kStages], kv_empty[S::kStages];
  __shared__ __align__(8) uint64_t s_full[2], p_full[2], drain_bar;
  __shared__ __align__(8) uint64_t last_full, last_clean;   // the causal tile's last V block
  __shared__ uint32_t tmem_slot;
  __shared__ int failed, drain_failed;
  // per slot: first and last key of any row, last first and first last key
  __shared__ int lo_key[2], hi_key[2], in_lo[2], in_hi[2];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(gtc_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ring = smem + 2 * S::kTile;
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
  const int p_tile = tile * (kSplit ? pps : 2 * pps);    // first position

  if (tid == 0) {
    mbar_init(&q_full, 1);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      lo_key[s] = INT_MAX;
      hi_key[s] = 0;
      in_lo[s] = 0;
      in_hi[s] = INT_MAX;
    }
    mbar_init(&drain_bar, 1);
    mbar_init(&last_full, 1);
    mbar_init(&last_clean, 1);
    failed = drain_failed = 0;
    mbar_init_fence();
  }
  // the kernel that joins the slices may start as SMs fall free
  if (!kCausal) asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if (warp == 9) tmem_alloc(&tmem_slot, 512);
  __syncthreads();
  int begin = 0, end = 0, position = -1;
  if (tid < 256) {
    const int slot = tid >> 7, r = tid & 127;
    const int p = p_tile + (kSplit ? 0 : slot * pps) + r / a.group;
    if (r < pps * a.group && p < a.positions) position = p;
    if (kCausal) {
      if (position >= 0) causal_range(a.offsets, a.sequences, position, begin, end);
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
    if (end > begin) {
      atomicMin(&lo_key[slot], begin);
      atomicMax(&hi_key[slot], end);
      atomicMax(&in_lo[slot], begin);
      atomicMin(&in_hi[slot], end);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
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
  const bool clear = end_row < GTC_KEYS;
  volatile int* gave_up = &failed;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
    if (warp == 8) {
      if (lane == 0 && (any0 || any1)) {   // TMA producer
        const int q_slots = kSplit ? 1 : 2;
        mbar_arrive_expect_tx(&q_full, q_slots * S::kBoxes * pps * a.group * S::kRow);
        for (int s = 0; s < q_slots; ++s)
          for (int b = 0; b < S::kBoxes; ++b)
            tma_load_3d(smem + s * S::kTile + b * S::kBox, &tm_q, b * 64, h * a.group,
                        p_tile + s * pps, &q_full);
        int g = 0;
        int armed[S::kStages] = {};
        bool last_armed = false;
        const auto load = [&](const CUtensorMap* map, int key, bool is_last = false) {
          const int st = g % S::kStages, r = g / S::kStages;
          if (*gave_up) return;
          if (r > 0 && !mbar_wait(&kv_empty[st], (r - 1) & 1)) {
            failed = 1;
            return;
          }
          uint64_t* bar = is_last ? &last_full : &kv_full[st];
          mbar_arrive_expect_tx(bar, S::kTile);
          for (int b = 0; b < S::kBoxes; ++b)
            tma_load_3d(ring + st * S::kTile + b * S::kBox, map, b * 64, h, key, bar);
          if (is_last) last_armed = true; else armed[st] = r + 1;
          ++g;
        };
        if (!kSplit) {
          for (int j = lo - 1; j < hi; ++j) {
            if (j >= lo) load(&tm_v, origin[0] + j * GTC_KEYS, clear && j == hi - 1);
            if (j + 1 < hi) load(&tm_k, origin[0] + (j + 1) * GTC_KEYS);
          }
        } else {
          for (int j = -1; j < hi; ++j)
            for (int s = 0; s < 2; ++s) {
              if (j >= 0 && j < last[s]) load(&tm_v, origin[s] + j * GTC_KEYS);
              if (j + 1 < last[s]) load(&tm_k, origin[s] + (j + 1) * GTC_KEYS);
            }
        }
        // every load in flight lands before the CTA exits
        if (!mbar_wait(&q_full, 0)) drain_failed = 1;
        if (last_armed && !mbar_wait(&last_full, 0)) drain_failed = 1;
        for (int s = 0; s < S::kStages; ++s)
          if (armed[s] > 0 && !mbar_wait(&kv_full[s], (armed[s] - 1) & 1)) drain_failed = 1;
      }
    } else if (warp == 9) {
      if (lane == 0) {                     // MMA issuer
        constexpr uint32_t i_qk = idesc_bf16_f32(128, GTC_KEYS);
        constexpr uint32_t i_pv = idesc_bf16_f32(128, DP) | IDESC_B_MN;
        constexpr int kPerBox = S::kRow / 32;             // 16-element steps of a box
        int g = 0;
        bool ok = any0 || any1;
        if (ok && !mbar_wait(&q_full, 0)) ok = false;
        const auto arrived = [&](int at) {
          if (ok && !mbar_wait(&kv_full[at % S::kStages], (at / S::kStages) & 1)) ok = false;
          tc_fence_after();
        };
        const auto scores = [&](int s, int at) {
          const uint64_t qd = smem_desc(smem + (kSplit ? 0 : s) * S::kTile, S::kRow, 16, 8 * S::kRow);
          const uint64_t kd = smem_desc(ring + (at % S::kStages) * S::kTile, S::kRow, 16,
                                        8 * S::kRow);
  #pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            const uint32_t off = ((kk / kPerBox) * S::kBox + (kk % kPerBox) * 32) >> 4;
            mma_bf16(tmem + s * GTC_KEYS, qd + off, kd + off, i_qk, kk > 0);
          }
          mma_commit(&s_full[s]);
        };
        const auto values = [&](int s, int at, int i) {
          if (ok && !mbar_wait(&p_full[s], i & 1)) ok = false;
          tc_fence_after();
          if (!ok) return;
          const uint64_t vd = smem_desc(ring + (at % S::kStages) * S::kTile, S::kRow, S::kBox,
                                        8 * S::kRow);
  #pragma unroll
          for (int kk = 0; kk < GTC_KEYS / 16; ++kk)
            mma_bf16_tmem_a(tmem + GTC_O + s * DP, tmem + s * GTC_KEYS + kk * 8,
                            vd + kk * ((16 * S::kRow) >> 4), i_pv, i > 0 || kk > 0);
          if (i == last[s] - first[s] - 1) mma_commit(&s_full[s]);
        };
        if (!kSplit) {
          for (int j = lo - 1; j < hi && ok; ++j) {
            const int gv = j >= lo ? g++ : -1, gk = j + 1 < hi ? g++ : -1;
            if (gv >= 0) {
              if (clear && j == hi - 1) {
                if (!mbar_wait(&last_clean, 0)) ok = false;
                tc_fence_after();
              } else {
                arrived(gv);
              }
            }
  #pragma unroll
            for (int s = 0; s < 2; ++s) {
              if (j >= first[s] && j < last[s]) values(s, gv, j - first[s]);
              if (s == 1 && gv >= 0 && ok) mma_commit(&kv_empty[gv % S::kStages]);
              if (s == 0 && gk >= 0) arrived(gk);
              if (ok && j + 1 >= first[s] && j + 1 < last[s]) scores(s, gk);
            }
            if (gk >= 0 && ok) mma_commit(&kv_empty[gk % S::kStages]);
          }
        } else {
          for (int j = -1; j < hi && ok; ++j)
  #pragma unroll
            for (int s = 0; s < 2; ++s) {
              if (j >= 0 && j < last[s]) {
                const int gv = g++;
                arrived(gv);
                values(s, gv, j);
                if (ok) mma_commit(&kv_empty[gv % S::kStages]);
              }
              if (j + 1 < last[s]) {
                const int gk = g++;
                arrived(gk);
                if (ok) {
                  scores(s, gk);
                  mma_commit(&kv_empty[gk % S::kStages]);
                }
              }
            }
        }
        if (!ok && (any0 || any1)) failed = 1;
        // no MMA may still use TMEM or shared memory when they are given back
        mma_commit(&drain_bar);
        if (!mbar_wait(&drain_bar, 0)) drain_failed = 1;
      }
    } else if (kCausal && warp == 10 && clear) {
      const int at = 1 + 2 * (hi - 1 - lo);   // its place in the ring
      // (the stream may still be a whole tile's work away from its last block)
      bool ok = false;
      while (!ok && !*gave_up) ok = mbar_wait_warp(&last_full, 0);
      if (ok) {
        uint8_t* block = ring + (at % S::kStages) * S::kTile;
        constexpr int kPieces = S::kRow / 16;
        for (int b = 0; b < S::kBoxes; ++b)
          for (int i = end_row * kPieces + lane; i < GTC_KEYS * kPieces; i += 32)
            *reinterpret_cast<uint4*>(block + b * S::kBox + i * 16) = make_uint4(0, 0, 0, 0);
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&last_clean);
      }
    }
  } else {                               // softmax and epilogue, one row per thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
    const int slot = warp >> 2;
    const int blocks = slot == 0 ? last[0] - first[0] : last[1] - first[1];
    const int key_first = slot == 0 ? origin[0] + first[0] * GTC_KEYS
                                    : origin[1] + first[1] * GTC_KEYS;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + slot * GTC_KEYS, t_o = tmem + lanes + GTC_O + slot * DP;
    const float c = a.scale_log2, slack = 8.f / c;
    const int all_from = in_lo[slot], all_to = in_hi[slot];
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < blocks; ++i) {
      if (!mbar_wait_warp(&s_full[slot], i & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t raw[4][32];
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_load32_async(t_s + 32 * q, raw[q]);
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_loaded32(raw[q]);
      if (negate) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int j = 0; j < 32; ++j) raw[q][j] ^= 0x80000000u;
      }
      const int key0 = key_first + i * GTC_KEYS;
      if (key0 < all_from || key0 + GTC_KEYS > all_to) {
        const int from = begin - key0, to = end - key0;
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (32 * q + j < from || 32 * q + j >= to) raw[q][j] = 0xff800000u;
      }
      float top = -INFINITY;
      {
        float t4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          t4[q] = __uint_as_float(raw[q][0]);
#pragma unroll
          for (int j = 1; j < 32; ++j) t4[q] = fmaxf(t4[q], __uint_as_float(raw[q][j]));
        }
        top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
      }
      if (i == 0) {
        m = top;
      } else {
        const bool grown = top > m + slack;
        if (__any_sync(0xffffffffu, grown)) {
          const float keep = grown ? gtc_exp2((m - top) * c) : 1.f;
          if (grown) m = top;
          l *= keep;
#pragma unroll
          for (int q = 0; q < DP / 32; ++q) {
            uint32_t o[32];
            tmem_load32_async(t_o + 32 * q, o);
            tmem_loaded32(o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
            tmem_store32(t_o + 32 * q, o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : m * c;
      const float2 c2 = make_float2(c, c), b2 = make_float2(-base, -base);
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t packed[32];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const uint32_t* s = raw[2 * half + q];
            float2 x = __ffma2_rn(make_float2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])),
                                  c2, b2);
            x.x = gtc_exp2(x.x);
            x.y = gtc_exp2(x.y);
            sum = __fadd2_rn(sum, x);
            packed[16 * q + j / 2] = gtc_pack(x.x, x.y);
          }
        tmem_store32(t_s + 32 * half, packed);
      }
      l += sum.x + sum.y;
      tmem_stored();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[slot]);
    }
    if (ok && blocks > 0 && !mbar_wait_warp(&s_full[slot], blocks & 1)) ok = false;
    if (!ok) failed = 1;
    tc_fence_after();

    const int r = tid & 127;
    const bool seen = end > begin && position >= 0;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if constexpr (kCausal) {
      // the output row goes through the slot's Q tile (its products are done)
      // so that whole rows leave in 16-byte pieces of neighbouring lanes
      constexpr int kPieces = DP / 8;
      uint8_t* stage = smem + slot * S::kTile;
      const auto piece = [&](int row, int at) {
        const int x = kPieces >= 8 ? row & 7 : (row >> 1) & 3;
        return reinterpret_cast<uint4*>(stage + row * (DP * 2) + ((at ^ x) << 4));
      };
      bool odd = seen && !(fabsf(l) <= FLT_MAX);
#pragma unroll 1
      for (int q = 0; q < DP / 32; ++q) {
        uint32_t o[32];
        if (blocks > 0) {
          tmem_load32_async(t_o + 32 * q, o);
          tmem_loaded32(o);
        }
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float x = seen ? __uint_as_float(o[j]) * inv : 0.f;
          big = fmaxf(big, x == x ? fabsf(x) : INFINITY);
          o[j] = __float_as_uint(x);
        }
        odd |= big == INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint4 w;
          w.x = gtc_pack(__uint_as_float(o[8 * k]), __uint_as_float(o[8 * k + 1]));
          w.y = gtc_pack(__uint_as_float(o[8 * k + 2]), __uint_as_float(o[8 * k + 3]));
          w.z = gtc_pack(__uint_as_float(o[8 * k + 4]), __uint_as_float(o[8 * k + 5]));
          w.w = gtc_pack(__uint_as_float(o[8 * k + 6]), __uint_as_float(o[8 * k + 7]));
          *piece(r, 4 * q + k) = w;
        }
      }
      __syncwarp();
      const int row0 = (warp & 3) * 32;
      const bool mine = position >= 0 && (seen || a.clear_rest);
      const unsigned write = __ballot_sync(0xffffffffu, mine && ok);
      unsigned again = __ballot_sync(0xffffffffu, odd && seen && ok);
#pragma unroll 1
      for (int i = 0; i < 32; i += 32 / kPieces) {
        const int rr = i + lane / kPieces, at = lane % kPieces;
        if (!((write >> rr) & 1) || at * 8 >= a.D) continue;
        const int row = row0 + rr;
        const int p = p_tile + slot * pps + row / a.group, head = h * a.group + row % a.group;
        *reinterpret_cast<uint4*>(a.out + (int64_t)p * a.o_sp + (int64_t)head * a.o_sh + at * 8) =
            *piece(row, at);
      }
      __syncwarp();
      while (again) {
        const int rr = __ffs(again) - 1, row = row0 + rr;
        again &= again - 1;
        causal_row_again<__nv_bfloat16, DP / 32>(
            a, p_tile + slot * pps + row / a.group, h * a.group + row % a.group,
            __shfl_sync(0xffffffffu, begin, rr), __shfl_sync(0xffffffffu, end, rr));
      }
    } else {
      const int part = kSplit ? 2 * slice + slot : slice;
      const int64_t at = ((int64_t)part * a.positions + position) * a.heads +
                         (int64_t)h * a.group + r % a.group;
#pragma unroll 1
      for (int q = 0; q < DP / 32; ++q) {
        uint32_t o[32];
        if (blocks > 0) {
          tmem_load32_async(t_o + 32 * q, o);
          tmem_loaded32(o);
        }
        if (position < 0 || !ok) continue;
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          if (32 * q + j >= a.D) break;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (blocks > 0)
            x = make_float4(__uint_as_float(o[j]) * inv, __uint_as_float(o[j + 1]) * inv,
                            __uint_as_float(o[j + 2]) * inv, __uint_as_float(o[j + 3]) * inv);
          *reinterpret_cast<float4*>(a.part + at * a.D + 32 * q + j) = x;
        }
      }
      if (position >= 0 && ok) a.part_lse[at] = l == 0.f ? -INFINITY : m * c + log2f(l);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
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
  using S = GtcShape<DP>;
  GroupedArgs<__nv_bfloat16> a = args;
  const int pps = 128 / a.group;                        // positions of a slot
  const int cols = S::kRow / 2;
  // a zero scale weighs every key alike; masked scores must stay -inf
  const int negate = a.scale_log2 < 0.f;
  a.scale_log2 = std::max(std::fabs(a.scale_log2), 1e-30f);
  CUtensorMap q, k, v;
  if (!gtc_map(&q, a.q, a.positions, a.heads, a.D, a.q_sp, a.q_sh, cols, a.group, pps) ||
      !gtc_map(&k, a.k, a.keys, a.kv_heads, a.D, a.k_st, a.k_sh, cols, 1, GTC_KEYS) ||
      !gtc_map(&v, a.v, a.keys, a.kv_heads, a.D, a.v_st, a.v_sh, cols, 1, GTC_KEYS))
    return GRS_ERR_SHAPE;
  const int64_t tiles = ((int64_t)a.positions + pps * (MODE == GTC_SPLIT ? 1 : 2) - 1) /
                        (pps * (MODE == GTC_SPLIT ? 1 : 2));
  if (tiles * a.kv_heads > INT_MAX || (MODE != GTC_CAUSAL && (a.kv_heads > 65535 ||
                                                              a.slices > 65535)))
    return GRS_ERR_SHAPE;
  const dim3 grid = MODE == GTC_CAUSAL
                        ? dim3((unsigned)(tiles * a.kv_heads))
                        : dim3((unsigned)tiles, a.kv_heads, a.slices);
  if (cudaFuncSetAttribute(grouped_tc_kernel<DP, MODE>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess)
    return GRS_ERR_CUDA;
  grouped_tc_kernel<DP, MODE><<<grid, GTC_THREADS, S::kSmem, counted(stream)>>>(q, k, v, a, pps,
                                                                               negate);
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
  return a.D <= 128 && a.group <= 128 &&
         gtc_rows_ok(a.q, a.positions, a.q_sp, a.heads, a.q_sh, a.D) &&
         gtc_rows_ok(a.k, a.keys, a.k_st, a.kv_heads, a.k_sh, a.D) &&
         gtc_rows_ok(a.v, a.keys, a.v_st, a.kv_heads, a.v_sh, a.D) &&
         (a.offsets == nullptr || gtc_rows_ok(a.out, a.positions, a.o_sp, a.heads, a.o_sh, a.D));
}

int grouped_tc_launch(const GroupedArgs<__nv_bfloat16>& a, cudaStream_t stream) {
  if (a.offsets) return gtc_width<GTC_CAUSAL>(a, stream);
  return grouped_tc_split(a.positions, a.group) ? gtc_width<GTC_SPLIT>(a, stream)
                                                : gtc_width<GTC_PAIR>(a, stream);
}

}  // namespace grs
