// Block bounds and block selection for the sparse decode: pa_block_bounds, pa_select_blocks.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/pa_decode.h"
#include "pa_block.h"
#include "pa_common.h"
#include "pa_launch.h"

namespace {

__device__ __forceinline__ int block_context(const PaBlockArgs& a, int b, int axis) {
  const int c = a.context_lens[b];
  return c < 0 ? 0 : (c > axis ? axis : c);
}

// ---- bounds -----------------------------------------------------------------------------------------------------------
//   lo_d = min_t k_td scale_t, hi_d = max_t k_td scale_t     over the block's tokens below the context length
//
// Read-bound: head size bytes per token and 4 D written per block; 64 sequences x 8 heads x 4096 tokens (332 MB) 66 us =
// 5.0 TB/s (one head per wave and exchanges through LDS: 77 us).  LPC lanes share a 16-byte chunk row of the block and
// take its tokens in turn (behind the last live token they take it again, which changes no extremum); every lane keeps
// [-lo, hi] of its chunk's head dims, so that all is maxima, and the lanes of a chunk row then halve what they hold with every
// exchange (a lane sends the half its partner keeps): 15 exchanges instead of 16 for each of log2(LPC) steps.
// FP8 codes are exact in 16-bit floats, where two maxima are one instruction (and a maximum passes over NaN); per-token
// scales need 32 bits.
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
enum { kBoundsFp8 = 0, kBoundsFp8Token = 1, kBoundsBf16 = 2 };

__device__ __forceinline__ uint32_t fp8x2_to_f16x2(uint32_t word, bool high_half) {
  union {
    f16x2 v;
    uint32_t u;
  } r;
  r.v = high_half ? __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, true))
                  : __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, false));
  return r.u;
}

template <int KIND>
struct BoundSlot;
// two head dims as 16-bit floats
template <>
struct BoundSlot<kBoundsFp8> {
  static constexpr int kDims = 2;
  uint32_t u = 0xfc00fc00u;  // -infinity
  __device__ __forceinline__ void take(uint32_t o) {
    const f16x2 x = __builtin_bit_cast(f16x2, u), y = __builtin_bit_cast(f16x2, o);
    u = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
  }
  __device__ __forceinline__ uint32_t bits() const { return u; }
  __device__ __forceinline__ float dim(int i) const { return (float)__builtin_bit_cast(f16x2, u)[i]; }
};
// one head dim in 32 bits
struct BoundSlot32 {
  static constexpr int kDims = 1;
  float x = -INFINITY;
  __device__ __forceinline__ void take(uint32_t o) { x = fmaxf(x, __uint_as_float(o)); }
  __device__ __forceinline__ uint32_t bits() const { return __float_as_uint(x); }
  __device__ __forceinline__ float dim(int) const { return x; }
};
template <>
struct BoundSlot<kBoundsFp8Token> : BoundSlot32 {};
template <>
struct BoundSlot<kBoundsBf16> : BoundSlot32 {};

// lane exchanges inside 16 lanes (DPP).  The pairs of a step need only differ in the bit that picks the half kept and, with the
// steps before, reach all lanes: 15 - i, then 7 - i, then the neighbour, then the next pair.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
constexpr int kDppSwap1 = 0xB1, kDppSwap2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140;

// one exchange: the lane keeps the upper or the lower half of its first 2 n slots
template <int CTRL, int N, typename Slot>
__device__ __forceinline__ void halve(Slot* slot, bool upper) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t keep = upper ? slot[N + i].bits() : slot[i].bits(), send = upper ? slot[i].bits() : slot[N + i].bits();
    Slot s;
    s.take(keep);
    s.take(dpp_u32<CTRL>(send));
    slot[i] = s;
  }
}

// SPLIT: the four waves of a workgroup share one (sequence, block, kv head) and meet in LDS (blocks of 64 tokens and more);
// otherwise a wave has kBoundsHeads kv heads of a (sequence, block) and asks for all of their keys before it looks at any:
// a wave with 2 KiB to read spends its time waiting for the context length, the table and the keys in turn.
constexpr int kBoundsHeads = 4;
// kv heads of a wave: fewer where a lane has more loads of a head in flight
template <int D, int KIND>
constexpr int bounds_heads() {
  return 16 / (64 / (D / (KIND == kBoundsBf16 ? 8 : 16))) > 2 ? kBoundsHeads / 2 : kBoundsHeads;
}

template <int D, int KIND, bool SPLIT>
__global__ __launch_bounds__(256) void pa_block_bounds_kernel(const PaBlockArgs a, const int axis, const int visits, const unsigned items) {
  typedef BoundSlot<KIND> Slot;
  constexpr bool FP8 = KIND != kBoundsBf16;
  constexpr int X = FP8 ? 16 : 8;
  constexpr int LPC = 64 / (D / X);         // lanes of a chunk row
  constexpr int HALF = X / Slot::kDims;     // slots of -lo, and as many of hi
  constexpr int KEEP = 2 * HALF / LPC;      // slots a lane is left with
  constexpr int U = 16 / LPC < 4 ? 16 / LPC : 4;  // loads in flight (a 16-token block has 16 / LPC for a lane)
  constexpr int HEADS = SPLIT ? 1 : bounds_heads<D, KIND>();
  static_assert(KEEP >= 1, "a lane is left with something");
  __shared__ uint32_t meet[SPLIT ? 3 : 1][SPLIT ? KEEP : 1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned item = SPLIT ? blockIdx.x : blockIdx.x * 4 + wave;
  if (item >= items) return;
  const unsigned head_groups = ((unsigned)a.num_kv_heads + HEADS - 1) / HEADS;
  const int h0 = (int)(item % head_groups) * HEADS;
  const unsigned visit = item / head_groups;
  const int b = (int)(visit / (unsigned)visits);
  const int bs = a.block_size;
  int ctx = sload_i32(a.context_lens + b);
  ctx = ctx > axis ? axis : ctx;
  const int first = a.new_tokens > 0 ? (ctx > a.new_tokens ? ctx - a.new_tokens : 0) / bs : 0;
  const int at = first + (int)(visit % (unsigned)visits);
  if (at >= (ctx + bs - 1) / bs) return;
  const int page = sload_i32(a.block_tables + (int64_t)b * a.stride_bt_s + at);
  if ((unsigned)page >= (unsigned)a.num_blocks) return;
  const int live = ctx - at * bs < bs ? ctx - at * bs : bs;
  const int heads = min(HEADS, a.num_kv_heads - h0);
  const char* kp = (const char*)a.key_cache + ((int64_t)page * a.stride_k_b + (int64_t)h0 * a.stride_k_h + (int64_t)(lane / LPC) * a.stride_k_c) * (FP8 ? 1 : 2);
  const int64_t kh = a.stride_k_h * (FP8 ? 1 : 2);
  const int64_t so = (int64_t)page * a.stride_kvscale_b + (int64_t)h0 * a.stride_kvscale_h;

  Slot slots[HEADS][2 * HALF];  // [-lo, hi]
  constexpr int kTurn = LPC * U * (SPLIT ? 4 : 1);
  for (int t0 = (SPLIT ? wave * LPC * U : 0) + lane % LPC; t0 - lane % LPC < live; t0 += kTurn) {
    u32x4 w[HEADS][U];
    float ts[HEADS][U];
#pragma unroll
    for (int g = 0; g < HEADS; ++g) {
      const int64_t gh = g < heads ? g : 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * LPC < live ? t0 + u * LPC : live - 1;
        w[g][u] = load16_stream(kp + gh * kh + t * 16);
        if constexpr (KIND == kBoundsFp8Token) ts[g][u] = a.key_scale[so + gh * a.stride_kvscale_h + t];
      }
    }
#pragma unroll
    for (int g = 0; g < HEADS; ++g) {
      Slot* slot = slots[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t word = w[g][u][i];
          if constexpr (KIND == kBoundsFp8) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t p = fp8x2_to_f16x2(word, e);
              slot[2 * i + e].take(p ^ 0x80008000u);
              slot[HALF + 2 * i + e].take(p);
            }
          } else if constexpr (KIND == kBoundsFp8Token) {
            const float x[4] = {__builtin_amdgcn_cvt_f32_fp8((int)word, 0) * ts[g][u], __builtin_amdgcn_cvt_f32_fp8((int)word, 1) * ts[g][u],
                                __builtin_amdgcn_cvt_f32_fp8((int)word, 2) * ts[g][u], __builtin_amdgcn_cvt_f32_fp8((int)word, 3) * ts[g][u]};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              slot[4 * i + e].take(__float_as_uint(-x[e]));
              slot[HALF + 4 * i + e].take(__float_as_uint(x[e]));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t x = e ? word & 0xffff0000u : word << 16;
              slot[2 * i + e].take(x ^ 0x80000000u);
              slot[HALF + 2 * i + e].take(x);
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int g = 0; g < HEADS; ++g) {
    if (g >= heads) break;
    Slot* slot = slots[g];
    // the lanes of a chunk row; `base` is where the slots that are left were
    int base = 0;
    const bool b3 = lane & 8, b2 = lane & 4, b1 = lane & 2, b0 = lane & 1;
    if constexpr (LPC == 16) {
      halve<kDppMirror, HALF>(slot, b3);
      halve<kDppHalfMirror, HALF / 2>(slot, b2);
      halve<kDppSwap1, HALF / 4>(slot, b0);
      halve<kDppSwap2, HALF / 8>(slot, b1);
      base = b3 * HALF + b2 * (HALF / 2) + b0 * (HALF / 4) + b1 * (HALF / 8);
    } else if constexpr (LPC == 8) {
      halve<kDppHalfMirror, HALF>(slot, b2);
      halve<kDppSwap1, HALF / 2>(slot, b0);
      halve<kDppSwap2, HALF / 4>(slot, b1);
      base = b2 * HALF + b0 * (HALF / 2) + b1 * (HALF / 4);
    } else if constexpr (LPC == 4) {
      halve<kDppSwap1, HALF>(slot, b0);
      halve<kDppSwap2, HALF / 2>(slot, b1);
      base = b0 * HALF + b1 * (HALF / 2);
    } else {
      static_assert(LPC == 2 || LPC == 4 || LPC == 8 || LPC == 16, "lanes of a chunk row");
      halve<kDppSwap1, HALF>(slot, b0);
      base = b0 * HALF;
    }
    if constexpr (SPLIT) {
      if (wave > 0) {
#pragma unroll
        for (int i = 0; i < KEEP; ++i) meet[wave - 1][i][lane] = slot[i].bits();
      }
      __syncthreads();
      if (wave > 0) return;
#pragma unroll
      for (int i = 0; i < KEEP; ++i) {
#pragma unroll
        for (int o = 0; o < 3; ++o) slot[i].take(meet[o][i][lane]);
      }
    }
    float scale = 1.f;
    if (a.kv_quant_mode == PA_QUANT_PER_TENSOR) scale = sload_f32(a.key_scale);
    if (a.kv_quant_mode == PA_QUANT_PER_BLOCK) scale = sload_f32(a.key_scale + so + g * a.stride_kvscale_h);
    const bool is_hi = base >= HALF;
    const float sign = is_hi ? scale : -scale;
    // (a negative scale turns the smallest code into the largest key)
    const bool row_hi = is_hi != (scale < 0.f);
    const float none = row_hi ? -INFINITY : INFINITY;  // a head dim without a key that is a number, whatever the scale (0 * infinity is NaN)
    __bf16* out = (__bf16*)a.bounds + (int64_t)page * a.stride_bounds_b + (int64_t)(h0 + g) * a.stride_bounds_h + (row_hi ? D : 0) +
                  lane / LPC * X + (is_hi ? base - HALF : base) * Slot::kDims;
    constexpr int N = KEEP * Slot::kDims;  // consecutive head dims
    uint32_t bits[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = slot[i / Slot::kDims].dim(i % Slot::kDims);
      bits[i] = __builtin_bit_cast(uint16_t, (__bf16)(x == -INFINITY ? none : x * sign));
    }
    if constexpr (N == 1) {
      *reinterpret_cast<uint16_t*>(out) = (uint16_t)bits[0];
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 2) *reinterpret_cast<uint32_t*>(out + i) = bits[i] | (bits[i + 1] << 16);
    }
  }
}

template <int D, int KIND>
int launch_bounds(const PaBlockArgs& a, int axis, int visits, hipStream_t s) {
  const int64_t most = (int64_t)a.num_seqs * visits * a.num_kv_heads;
  if (most > 0x7fffffffLL) return PA_ERR_BAD_SHAPE;
  if (a.block_size > 16) return pa_launch(pa_block_bounds_kernel<D, KIND, true>, dim3((unsigned)most), dim3(256), 0, s, a, axis, visits, (unsigned)most);
  const int heads = bounds_heads<D, KIND>();
  const int64_t items = (int64_t)a.num_seqs * visits * ((a.num_kv_heads + heads - 1) / heads);
  return pa_launch(pa_block_bounds_kernel<D, KIND, false>, dim3((unsigned)((items + 3) / 4)), dim3(256), 0, s, a, axis, visits, (unsigned)items);
}

template <int D>
int launch_bounds(const PaBlockArgs& a, int axis, int visits, hipStream_t s) {
  if (a.kv_dtype == PA_DTYPE_BF16) return launch_bounds<D, kBoundsBf16>(a, axis, visits, s);
  if (a.kv_quant_mode == PA_QUANT_PER_TOKEN) return launch_bounds<D, kBoundsFp8Token>(a, axis, visits, s);
  return launch_bounds<D, kBoundsFp8>(a, axis, visits, s);
}

// ---- scores ------------------------------------------------------------------------------------------------------------
//   score(block) = max over rows r of x_r,   x_r = sum_d q+_rd hi_d + q-_rd lo_d      (q+ = max(q, 0), q- = min(q, 0))
//
// The ranking is by the scores' values in 64 bits, but almost every block is decided by less.  pa_block_score_kernel forms
// s_r = x_r in 32 bits on v_mfma_f32_16x16x32_bf16 (blocks are the rows, query rows the columns, [lo, hi] against [q-, q+] the
// 2 D reduction indices) and, with the sign bits cleared, a_r = sum of the terms' magnitudes.  The terms are exact in 32 bits;
// a sum of 2 D of them in any order, rounded or cut at every step, is off by at most 2 D 2^-23 a_r, so the score lies
// within e = max_r (2 D 2^-23 a_r) of s = max_r s_r.  The workspace holds (s, e) of every block; e = infinity says that the
// 32-bit sums decide nothing (an infinity or NaN among them, or a table entry outside the cache).
// Read-bound: 4 D bytes per block and head against 2 * 2 D / 32 MFMAs per 16 of them; 4 sequences x 8 heads x 8192 blocks
// (134 MB) 32 us = 4.2 TB/s, 64 x 8 x 256 blocks 14 us (every sum in 64 bits on the vector ALU: 331 and 128 us).
struct BlockScore {
  float s, e;
};

// the maximum over a row of 16 lanes
__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, __uint_as_float(dpp_u32<kDppSwap1>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(dpp_u32<kDppSwap2>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(dpp_u32<kDppHalfMirror>(__float_as_uint(v))));
  return fmaxf(v, __uint_as_float(dpp_u32<kDppMirror>(__float_as_uint(v))));
}

constexpr int kScoreWaves = 4;

// [lo, hi] against [q-, q+] of one 16-row tile as MFMA operands: operand c of lane l at (c * 64 + l) * 16 bytes
template <int D>
__device__ __forceinline__ void stage_query(const PaBlockArgs& a, int b, int h, int rows_valid, int tiles, u32x4* q_lds, int tid, int threads) {
  constexpr int KM = D / 32;
  const int Ge = a.q_len * a.group_size;
  for (int i = tid; i < tiles * KM * 64; i += threads) {
    const int l = i & 63, c = (i >> 6) % KM, tile = i / (64 * KM);
    const int row = 16 * tile + (l & 15);
    u32x4 q = {0, 0, 0, 0};
    if (row < rows_valid)
      q = load16((const __bf16*)a.query + (int64_t)b * a.stride_q_s + (int64_t)(h * Ge + row) * a.stride_q_h + 32 * c + 8 * (l >> 4));
    u32x4 neg, pos;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // (a NaN goes to both sides; -0 is 0 on either)
      const uint32_t lo = q[w] & 0xffffu, hi = q[w] >> 16;
      const uint32_t lo_neg = lo >> 15, hi_neg = hi >> 15, lo_nan = (lo & 0x7fffu) > 0x7f80u, hi_nan = (hi & 0x7fffu) > 0x7f80u;
      neg[w] = (lo_neg | lo_nan ? lo : 0u) | (hi_neg | hi_nan ? hi << 16 : 0u);
      pos[w] = (!lo_neg | lo_nan ? lo : 0u) | (!hi_neg | hi_nan ? hi << 16 : 0u);
    }
    q_lds[(tile * 2 * KM + c) * 64 + l] = neg;
    q_lds[(tile * 2 * KM + KM + c) * 64 + l] = pos;
  }
}

// One wave scores 16 blocks (blocks at .. at + 15 of the sequence, those below `end`) and writes them at out[at ..].
template <int D>
struct ScoreTile {
  static constexpr int KM = D / 32;
  u32x4 box[2 * KM];
  bool ok;
  __device__ __forceinline__ void load(const PaBlockArgs& a, const int* table, int h, int at, int end, int lane) {
    const int i = at + (lane & 15);
    const int page = i < end ? table[i] : 0;
    ok = (unsigned)page < (unsigned)a.num_blocks;
    const __bf16* p = (const __bf16*)a.bounds + (int64_t)(ok ? page : 0) * a.stride_bounds_b + (int64_t)h * a.stride_bounds_h + 8 * (lane >> 4);
#pragma unroll
    for (int c = 0; c < 2 * KM; ++c) box[c] = load16(p + 32 * c);  // (two loads share each 128-byte line: it has to stay in the cache)
  }
  __device__ __forceinline__ void score(const u32x4* q_lds, int tiles, int rows_valid, BlockScore* out, int at, int end, int lane) const {
    constexpr float kBound = 2 * D * 0x1p-23f;
    const int li = lane & 15, kg = lane >> 4;
    f32x4 best = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, off = {0.f, 0.f, 0.f, 0.f};
    for (int tile = 0; tile < tiles; ++tile) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f}, m = s;
#pragma unroll
      for (int c = 0; c < 2 * KM; ++c) {
        Bf16x8Bits x, q, xa, qa;
        x.u = box[c];
        q.u = q_lds[(tile * 2 * KM + c) * 64 + lane];
        xa.u = x.u & 0x7fff7fffu;
        qa.u = q.u & 0x7fff7fffu;
        s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, q.v, s, 0, 0, 0);
        m = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xa.v, qa.v, m, 0, 0, 0);
      }
      if (16 * tile + li < rows_valid) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          best[r] = fmaxf(best[r], s[r]);
          // (infinite or NaN magnitudes: no bound)
          off[r] = m[r] < 0x1p126f ? fmaxf(off[r], m[r] * kBound + 0x1p-100f) : INFINITY;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      best[r] = row16_max(best[r]);
      off[r] = row16_max(off[r]);
    }
    // lane group kg holds blocks 4 kg .. 4 kg + 3; lane li < 4 of it writes block 4 kg + li (the entry that lane loaded: 4 kg + li)
    const bool entry_ok = __shfl((int)ok, 4 * kg + (li & 3));
    const int i = at + 4 * kg + li;
    if (li < 4 && i < end) {
      BlockScore v;
      v.s = li == 0 ? best[0] : li == 1 ? best[1] : li == 2 ? best[2] : best[3];
      v.e = li == 0 ? off[0] : li == 1 ? off[1] : li == 2 ? off[2] : off[3];
      if (!entry_ok || !(v.s > -INFINITY)) v.e = INFINITY;
      out[i] = v;
    }
  }
};

// grid: (stretches of `chunk` blocks, a multiple of 64) x (sequence, kv head)
template <int D>
__global__ __launch_bounds__(64 * kScoreWaves) void pa_block_score_kernel(const PaBlockArgs a, const int axis, const int axis_blocks, const int chunk) {
  extern __shared__ __attribute__((aligned(16))) u32x4 q_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunks = (axis_blocks + chunk - 1) / chunk;
  const int h = (int)(blockIdx.x % (unsigned)a.num_kv_heads);
  const unsigned at_chunk = blockIdx.x / (unsigned)a.num_kv_heads;
  const int b = (int)(at_chunk / (unsigned)chunks);
  const int begin = (int)(at_chunk % (unsigned)chunks) * chunk;
  const int nb = (block_context(a, b, axis) + a.block_size - 1) / a.block_size;
  const int end = min(begin + chunk, nb - a.recent_blocks);
  if (nb <= a.num_selected || begin >= end) return;  // (every block is taken, or these blocks are: nobody reads their scores)
  int qb = a.q_lens ? a.q_lens[b] : a.q_len;
  qb = qb < 0 ? 0 : (qb > a.q_len ? a.q_len : qb);
  const int rows_valid = qb * a.group_size, tiles = (rows_valid + 15) / 16;
  const int* table = a.block_tables + (int64_t)b * a.stride_bt_s;
  BlockScore* out = (BlockScore*)a.workspace + ((int64_t)b * a.num_kv_heads + h) * axis_blocks;
  ScoreTile<D> t;
  int at = begin + 16 * wave;
  if (at < end) t.load(a, table, h, at, end, lane);
  stage_query<D>(a, b, h, rows_valid, tiles, q_lds, threadIdx.x, 64 * kScoreWaves);
  __syncthreads();
  for (; at < end; at += 16 * kScoreWaves) {
    const ScoreTile<D> now = t;
    if (at + 16 * kScoreWaves < end) t.load(a, table, h, at + 16 * kScoreWaves, end, lane);
    now.score(q_lds, tiles, rows_valid, out, at, end, lane);
  }
}

// a score as a key whose unsigned order is the scores' order
__device__ __forceinline__ unsigned long long score_key(double s) {
  s = s + 0.0;  // -0 and +0 are equal scores
  const unsigned long long u = (unsigned long long)__double_as_longlong(s);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// The key of one block's score in 64 bits, by one wave: 8 rows at a time, 8 lanes to a row, 8 head dims of D to a lane and
// turn.  Products of bf16 numbers have 16 significant bits and D of them grow by log2(D) more, so a sum is exact while its terms
// are no more than 53 - 16 - log2(D) binary orders apart (29 at D = 256).  Beyond that it is a 64-bit sum in this one order: the
// same for equal bounds, whichever wave forms it.
__device__ __forceinline__ unsigned long long exact_key(const PaBlockArgs& a, int b, int h, int page, int rows_valid, int lane) {
  double best = -INFINITY;
  if ((unsigned)page < (unsigned)a.num_blocks) {
    const int D = a.head_size, Ge = a.q_len * a.group_size;
    const __bf16* box = (const __bf16*)a.bounds + (int64_t)page * a.stride_bounds_b + (int64_t)h * a.stride_bounds_h;
    for (int row0 = 0; row0 < rows_valid; row0 += 8) {
      const int row = row0 + (lane >> 3);
      const __bf16* q = (const __bf16*)a.query + (int64_t)b * a.stride_q_s + (int64_t)(h * Ge + (row < rows_valid ? row : row0)) * a.stride_q_h;
      double s = 0.0;
      for (int d = 8 * (lane & 7); d < D; d += 64) {
        const u32x4 x = load16(q + d), lo = load16(box + d), hi = load16(box + D + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int sh = 16 * (e & 1);
          const float qe = bf16_bits_to_f32((x[e >> 1] >> sh) & 0xffffu);
          const double l = (double)bf16_bits_to_f32((lo[e >> 1] >> sh) & 0xffffu), u = (double)bf16_bits_to_f32((hi[e >> 1] >> sh) & 0xffffu);
          s += (double)(qe < 0.f ? 0.f : qe) * u + (double)(qe > 0.f ? 0.f : qe) * l;  // (0 * infinity is NaN in either)
        }
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) s += __shfl_xor(s, o);
      if (s == INFINITY) s = 0x1.fffffffffffffp1023;  // (below the blocks that are always taken)
      if (row < rows_valid && s > best) best = s;     // (a NaN is passed over)
    }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) {
      const double t = __shfl_xor(best, o);
      if (t > best) best = t;
    }
  }
  return score_key(best);
}

// ---- selection -----------------------------------------------------------------------------------------------------------
// One workgroup per (sequence, kv head).  The blocks are counted into kBins equal intervals of s; the one in which the count
// from above reaches `want` holds the threshold, up to the errors e.  Blocks that are above it by more than the
// errors are taken, blocks below it by more are not, and the few between (the candidates) are ranked by their scores in
// 64 bits.  Bound by latency, not by bytes (8 per block, from L2): 5 us for 128 blocks, 8 us for 512 lists of 256, 15 us for 32
// of 8192 (eight byte passes over 64-bit keys: 68, 88 and 108 us).
//
// The workgroup forms EVERY score of its list in 64 bits, one block per wave at a time, and finds the threshold by eight passes
// over the keys' bytes, when
//   * a list has more than 32 kFlagWords = 65536 blocks;
//   * one of its scores is not bounded by 32 bits (e = infinity): a bound that is infinite or NaN, a table entry outside the
//     cache, or a sequence without a query row;
//   * more than kCandidates blocks are left between: many equal blocks, or one whose keys are far larger than the others', which
//     widens all bins and the list's largest error E.
// The list is the same, the time is not: 32 lists of 8192 blocks, scores and selection together, 44 us for 256 of them, 74 with
// one block of 30 times the keys, 2.0 ms with one of 100 times (1024 of them: 48 us, 146 us, 2.0 ms), 2.0 ms with one bad entry;
// 8 lists of 65536 blocks 116 us, of 65537 16 ms.  The blocks that are always taken are not among the scores: first_blocks = 1
// spares a list its first block's large keys.
constexpr int kSelectThreads = 512;
constexpr int kAhead = 4;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kBins = 2048;
constexpr int kCandidates = 512;
constexpr int kFlagWords = 2048;  // 32 blocks each

// exclusive prefix sum of x over the workgroup and its total
__device__ __forceinline__ int workgroup_scan(int x, int* wave_sums, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(s, d);
    if (lane >= d) s += y;
  }
  __syncthreads();
  if (lane == 63) wave_sums[wave] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    const int v = wave_sums[w];
    before += w < wave ? v : 0;
    total += v;
  }
  return before + s - x;
}

__global__ __launch_bounds__(kSelectThreads) void pa_block_select_kernel(const PaBlockArgs a, const int axis, const int axis_blocks) {
  __shared__ int hist[kBins];
  __shared__ uint32_t flags[kFlagWords];
  __shared__ unsigned long long cand_key[kCandidates];
  __shared__ int cand[kCandidates];
  __shared__ int wave_sums[kSelectWaves];
  __shared__ float red[4][kSelectWaves];
  __shared__ int found[2], num_cand, num_in;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = (int)(blockIdx.x % (unsigned)a.num_kv_heads), b = (int)(blockIdx.x / (unsigned)a.num_kv_heads);
  const int nb = (block_context(a, b, axis) + a.block_size - 1) / a.block_size;
  const int K = a.num_selected;
  int32_t* out = a.selected_blocks + (int64_t)b * a.stride_sel_s + (int64_t)h * a.stride_sel_h;
  const int count = nb < K ? nb : K;
  if (tid == 0) a.selected_counts[(int64_t)b * a.stride_cnt_s + h] = count;
  for (int i = count + tid; i < K; i += kSelectThreads) out[i] = -1;
  if (nb <= K) {
    for (int i = tid; i < nb; i += kSelectThreads) out[i] = i;
    return;
  }
  // blocks [begin, end) have scores; `want` of them are taken (nb > K >= first + recent: the two ends do not meet)
  const int begin = a.first_blocks, end = nb - a.recent_blocks;
  const int want = K - a.first_blocks - a.recent_blocks;
  int qb = a.q_lens ? a.q_lens[b] : a.q_len;
  qb = qb < 0 ? 0 : (qb > a.q_len ? a.q_len : qb);
  const int rows_valid = qb * a.group_size;
  const int* table = a.block_tables + (int64_t)b * a.stride_bt_s;
  const BlockScore* score = (const BlockScore*)a.workspace + (int64_t)blockIdx.x * axis_blocks;

  bool by_32 = nb <= 32 * kFlagWords;
  if (by_32 && want > 0) {
    // ---- range of s, largest e ----------------------------------------------------------------------------------------
    float mn = INFINITY, mx = -INFINITY, E = 0.f;
    // (kAhead scores of a thread are asked for at a time: one by one a pass would be a chain of L2 latencies; behind the end
    // the last one is read again)
    for (int i0 = begin + tid; i0 < end; i0 += kAhead * kSelectThreads) {
      BlockScore v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) v[u] = score[min(i0 + u * kSelectThreads, end - 1)];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        mn = fminf(mn, v[u].s);
        mx = fmaxf(mx, v[u].s);
        E = fmaxf(E, v[u].e);
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      mn = fminf(mn, __shfl_xor(mn, o));
      mx = fmaxf(mx, __shfl_xor(mx, o));
      E = fmaxf(E, __shfl_xor(E, o));
    }
    if (lane == 0) {
      red[0][wave] = mn;
      red[1][wave] = mx;
      red[2][wave] = E;
    }
    for (int i = tid; i < kBins; i += kSelectThreads) hist[i] = 0;
    if (tid == 0) num_cand = num_in = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelectWaves; ++w) {
      mn = fminf(mn, red[0][w]);
      mx = fmaxf(mx, red[1][w]);
      E = fmaxf(E, red[2][w]);
    }
    by_32 = E < INFINITY;
    if (by_32) {
      // a monotone map of the scores to bins (a range that overflows puts everything into bin 0)
      const float scale = mx - mn > 0.f ? (float)(kBins - 1) / (mx - mn) : 0.f;
      auto bin = [&](float s) {
        const float x = (s - mn) * scale;
        return x >= (float)(kBins - 1) ? kBins - 1 : (x > 0.f ? (int)x : 0);
      };
      for (int i0 = begin + tid; i0 < end; i0 += kAhead * kSelectThreads) {
        float v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = score[min(i0 + u * kSelectThreads, end - 1)].s;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (i0 + u * kSelectThreads < end) atomicAdd(&hist[bin(v[u])], 1);
      }
      __syncthreads();
      // the bin in which the count from above reaches `want`: a thread owns four bins, the highest first
      constexpr int kOwn = kBins / kSelectThreads;
      int own[kOwn], sum = 0, total;
#pragma unroll
      for (int k = 0; k < kOwn; ++k) sum += own[k] = hist[kBins - 1 - (kOwn * tid + k)];
      int before = workgroup_scan(sum, wave_sums, total);
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        if (before < want && before + own[k] >= want) found[0] = kBins - 1 - (kOwn * tid + k);
        before += own[k];
      }
      __syncthreads();
      const int edge = found[0];
      // ---- taken, candidate or neither: a wave looks at 64 consecutive blocks ----------------------------------------------
      int taken = 0;
      for (int j0 = 64 * wave; j0 < nb; j0 += 64 * kSelectWaves * kAhead) {
        BlockScore v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i = j0 + 64 * kSelectWaves * u + lane;
          v[u] = score[i < begin ? begin : min(i, end - 1)];
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i0 = j0 + 64 * kSelectWaves * u, i = i0 + lane;
          if (i0 >= nb) break;
          // (s +- (e + E), with room for the roundings here: e is at least 2^-16 of |s|)
          const float slack = (v[u].e + E) * 1.01f;
          const bool scored = i >= begin && i < end;
          const bool in = scored && bin(v[u].s - slack) > edge;
          const uint64_t above = __builtin_amdgcn_ballot_w64(in), ends = __builtin_amdgcn_ballot_w64(i < nb && !scored);
          taken += __builtin_popcountll(above);
          if (lane < 2) flags[(i0 >> 5) + lane] = (uint32_t)((above | ends) >> (32 * lane));
          if (scored && !in && bin(v[u].s + slack) >= edge) {
            const int at = atomicAdd(&num_cand, 1);
            if (at < kCandidates) cand[at] = i;
          }
        }
      }
      if (lane == 0 && taken) atomicAdd(&num_in, taken);
      __syncthreads();
      by_32 = num_cand <= kCandidates;
    }
    if (by_32) {
      const int n = num_cand, take = want - num_in;
      if (take < n) {
        for (int c = wave; c < n; c += kSelectWaves) {
          const unsigned long long k = exact_key(a, b, h, table[cand[c]], rows_valid, lane);
          if (lane == 0) cand_key[c] = k;
        }
      }
      __syncthreads();
      for (int c = tid; c < n; c += kSelectThreads) {
        const unsigned long long k = cand_key[c];
        const int at = cand[c];
        int rank = 0;
        if (take < n)
          for (int o = 0; o < n; ++o) rank += cand_key[o] > k || (cand_key[o] == k && cand[o] < at);
        if (rank < take) atomicOr(&flags[at >> 5], 1u << (at & 31));
      }
      __syncthreads();
    }
  } else if (by_32) {
    for (int i0 = 64 * wave; i0 < nb; i0 += 64 * kSelectWaves) {
      const int i = i0 + lane;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(i < nb && (i < begin || i >= end));
      if (lane < 2) flags[(i0 >> 5) + lane] = (uint32_t)(mask >> (32 * lane));
    }
    __syncthreads();
  }
  if (by_32) {
    // the flags' blocks in ascending order
    const int words = (nb + 31) >> 5;
    int done = 0;
    for (int w0 = 0; w0 < words; w0 += kSelectThreads) {
      uint32_t f = w0 + tid < words ? flags[w0 + tid] : 0;
      int total;
      int at = done + workgroup_scan(__builtin_popcount(f), wave_sums, total);
      done += total;
      while (f) {
        out[at++] = 32 * (w0 + tid) + __builtin_ctz(f);
        f &= f - 1;
      }
    }
    return;
  }

  // ---- every score in 64 bits ----------------------------------------------------------------------------------------------
  unsigned long long* key = (unsigned long long*)a.workspace + (int64_t)blockIdx.x * axis_blocks;
  __syncthreads();  // everybody is done with the 32-bit scores
  for (int i = begin + wave; i < end; i += kSelectWaves) {
    const unsigned long long k = exact_key(a, b, h, table[i], rows_valid, lane);
    if (lane == 0) key[i] = k;
  }
  __threadfence_block();
  __syncthreads();
  unsigned long long prefix = 0;
  int left = want;  // of the keys that share the digits fixed so far, how many are still to be taken
  for (int shift = 56; shift >= 0 && want > 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    for (int i = begin + tid; i < end; i += kSelectThreads) {
      const unsigned long long k = key[i];
      if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    int total;
    const int mine = tid < 256 ? hist[255 - tid] : 0;
    const int before = workgroup_scan(mine, wave_sums, total);
    if (tid < 256 && before < left && before + mine >= left) {
      found[0] = 255 - tid;
      found[1] = before;
    }
    __syncthreads();
    prefix |= (unsigned long long)found[0] << shift;
    left -= found[1];
  }
  // the blocks at the ends, the keys above the threshold, and the first `left` that equal it
  int done = 0, equal_before = 0;
  for (int i0 = 0; i0 < nb; i0 += kSelectThreads) {
    const int i = i0 + tid;
    const bool scored = i >= begin && i < end;
    const unsigned long long k = scored && want > 0 ? key[i] : 0;
    const bool eq = scored && want > 0 && k == prefix;
    int total;
    const int rank = equal_before + workgroup_scan(eq, wave_sums, total);
    equal_before += total;
    const bool take = i < nb && (!scored || (want > 0 && (k > prefix || (eq && rank < left))));
    const int at = done + workgroup_scan(take, wave_sums, total);
    done += total;
    if (take) out[at] = i;
  }
}

int check_bounds(const PaBlockArgs* a) {
  if (int rc = check_block_sizes(a)) return rc;
  if (int rc = check_block_cache(a, false)) return rc;
  if (!a->bounds) return PA_ERR_NULL_POINTER;
  if (a->new_tokens < 0 || !block_aligned16(a->bounds) || a->stride_bounds_b % 8 || a->stride_bounds_h % 8) return PA_ERR_BAD_SHAPE;
  return PA_OK;
}

int check_select(const PaBlockArgs* a) {
  if (int rc = check_block_sizes(a)) return rc;
  if (int rc = check_block_rows(a)) return rc;
  if (!a->bounds || !a->query || !a->selected_blocks || !a->selected_counts) return PA_ERR_NULL_POINTER;
  if (!block_aligned16(a->bounds) || a->stride_bounds_b % 8 || a->stride_bounds_h % 8) return PA_ERR_BAD_SHAPE;
  if (!block_aligned16(a->query) || a->stride_q_s % 8 || a->stride_q_h % 8) return PA_ERR_BAD_SHAPE;
  if (a->num_selected <= 0 || a->first_blocks < 0 || a->recent_blocks < 0 ||
      (int64_t)a->first_blocks + a->recent_blocks > a->num_selected)
    return PA_ERR_BAD_SHAPE;
  return PA_OK;
}

int axis_blocks_of(const PaBlockArgs& a) {
  const int n = (block_axis(a) + a.block_size - 1) / a.block_size;
  return n > 0 ? n : 1;
}

}  // namespace

extern "C" {

int pa_block_bounds(const PaBlockArgs* a, void* hip_stream) {
  if (int rc = check_bounds(a)) return rc;
  hipStream_t stream = reinterpret_cast<hipStream_t>(hip_stream);
  const int axis = block_axis(*a);
  int visits = axis_blocks_of(*a);
  if (a->new_tokens > 0) {
    const int64_t reach = ((int64_t)a->new_tokens + a->block_size - 2) / a->block_size + 1;
    if (reach < visits) visits = (int)reach;
  }
  return a->head_size == 64    ? launch_bounds<64>(*a, axis, visits, stream)
         : a->head_size == 128 ? launch_bounds<128>(*a, axis, visits, stream)
                               : launch_bounds<256>(*a, axis, visits, stream);
}

int64_t pa_select_blocks_workspace_bytes(const PaBlockArgs* a) {
  if (int rc = check_select(a)) return rc;
  return (int64_t)a->num_seqs * a->num_kv_heads * axis_blocks_of(*a) * 8;
}

int pa_select_blocks(const PaBlockArgs* a, void* hip_stream) {
  const int64_t need = pa_select_blocks_workspace_bytes(a);
  if (need < 0) return (int)need;
  if (!a->workspace) return PA_ERR_NULL_POINTER;
  if (a->workspace_bytes < need || !block_aligned16(a->workspace)) return PA_ERR_SCRATCH_TOO_SMALL;
  hipStream_t stream = reinterpret_cast<hipStream_t>(hip_stream);
  const int axis = block_axis(*a), blocks = axis_blocks_of(*a);
  const int64_t heads = (int64_t)a->num_seqs * a->num_kv_heads;
  // stretches long enough to pay for staging the query, short enough to fill the GPU: 64 blocks up to 512 workgroups
  int64_t chunk = (heads * blocks / 512 + 63) / 64 * 64;
  chunk = chunk < 64 ? 64 : (chunk > 1024 ? 1024 : chunk);
  const int64_t grid = heads * ((blocks + chunk - 1) / chunk);
  if (grid > 0x7fffffffLL) return PA_ERR_BAD_SHAPE;
  const dim3 g((unsigned)grid), t(64 * kScoreWaves);
  const unsigned lds = (unsigned)((a->q_len * a->group_size + 15) / 16) * a->head_size * 64;  // [q-, q+] of 16 rows: 64 D bytes
  const int rc = a->head_size == 64    ? pa_launch(pa_block_score_kernel<64>, g, t, lds, stream, *a, axis, blocks, (int)chunk)
                 : a->head_size == 128 ? pa_launch(pa_block_score_kernel<128>, g, t, lds, stream, *a, axis, blocks, (int)chunk)
                                       : pa_launch(pa_block_score_kernel<256>, g, t, lds, stream, *a, axis, blocks, (int)chunk);
  if (rc) return rc;
  return pa_launch(pa_block_select_kernel, dim3((unsigned)heads), dim3(kSelectThreads), 0, stream, *a, axis, blocks);
}

}  // extern "C"
