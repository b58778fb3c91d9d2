// Decode attention at the granularity of cache blocks: pa_block_attention.
//
//   out[row] = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q.k_t - max),   over the tokens of the selected blocks
//
// One pass over K and V with a running maximum and sum.  A workgroup of four waves owns one (sequence, stretch of the
// token axis, kv head, group of NT 16-row query tiles); its waves take the stretch's steps of 64 tokens in turn and merge
// in LDS.  The token axis is the list of selected blocks (all blocks without a list), so a step is four 16-token pieces
// of blocks wherever they lie.  With a cut axis the workgroups leave (max, sum, O) in f32 and a second kernel merges.
//
// v_mfma_f32_16x16x32_bf16 holds, in lane l (li = l % 16, kg = l / 16), eight consecutive reduction indices of row /
// column li of its operands and rows 4 kg .. 4 kg + 3 of column li of its result.
//   S^T[token, row] = K Q^T   tile j takes tokens 4 j .. 4 j + 3 of EVERY piece (its row i: piece i / 4, token 4 j + i % 4), so
//                             lane group kg ends up with the logits of all 16 tokens of piece kg, and P never moves
//                             between lanes.  A lane's 16-byte load is 16 (FP8) or 8 (bf16) head dims of one token.
//   O^T[dim, row]  += V^T P   MFMA u takes tokens 8 u .. 8 u + 7 of every piece: A is half of the 16 bytes (FP8) that hold the
//                             16 tokens of head dim li of a 16-dim row, B the eight probabilities the lane has.
// FP8 codes are exact in bf16, and so are their products with powers of two; q is bf16; P is carried as two bf16 terms
// (p = hi + lo, 16 significant bits): a product has no rounding that the f32 accumulator would not have.  The scale of a block
// is a factor of the lane's logits (K); V's goes into the conversion of the codes (its power of two) and into the exponents
// (the rest): one load each per step and lane.
//
// Bound by the read of the cache up to 16 query rows per kv head: 64 sequences x 8 heads x 4096 tokens (537 MB) 89 us = 6.0
// TB/s, 4 x 8 x 131072 tokens 180 us = 6.0 TB/s (a 4 GiB copy reaches 4.8); the first of these with a bf16 cache 5.9 TB/s, with
// head size 64 5.7 and 256 6.2, in blocks of 64 and 1024 tokens 5.5 and 5.2, with per-token scales 4.5 (head size 256: 3.7, the
// registers spill).  A wave has a whole step of K and V in flight, two waves per SIMD.  17 .. 32 rows 104 us.  Three and more
// tiles (33 .. 64 rows) are bound by the vector ALU, some 350 instructions per tile and step around 48 MFMAs (32 ragged sequences of
// up to 8191 tokens, 64 rows: 111 us); two tiles per workgroup beat one (144 us with the merge against 125) and four (168: the
// registers spill).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/pa_decode.h"
#include "pa_block.h"
#include "pa_common.h"
#include "pa_launch.h"

namespace {

constexpr int kBlockWaves = 4;
enum { kScaleOne = 0, kScaleToken = 1, kScaleBlock = 2 };  // one factor per call (or none) / per token / per block

// What the host decides about a call; the kernels read it beside the caller's arguments.
struct BlockCut {
  int axis;        // tokens of the longest context (without a list)
  int part;        // tokens of the axis that a workgroup takes, a multiple of 256
  int parts;       // workgroups along the axis
  int row_groups;  // workgroups along the query rows
  int spread;      // 1: the kv heads of a (sequence, stretch) go to different XCDs, 0: they share one
};

__device__ __forceinline__ float fast_log2(float x) { return __builtin_amdgcn_logf(x); }

// tokens on the (virtual) axis of a (sequence, head)
__device__ __forceinline__ int virtual_tokens(const PaBlockArgs& a, int b, int h, int ctx) {
  if (!a.selected_blocks) return ctx;
  int n = a.selected_counts ? sload_i32(a.selected_counts + (int64_t)b * a.stride_cnt_s + h) : a.num_selected;
  n = n < 0 ? 0 : (n > a.num_selected ? a.num_selected : n);
  return ctx > 0 ? n * a.block_size : 0;
}

// STEP: tokens a wave takes at a time, 64 or 32 (half the registers in flight: head size 256, 16-bit caches, and two tiles with
// per-token scales at head size 128).  A lane group holds the STEP / 4 consecutive tokens kg * STEP / 4 .. of it, the whole or
// the half of a 16-token piece.
// Q_LDS: the query operands wait in LDS (the same for the four waves) and not in registers.
// OCC: waves per SIMD that the registers are cut for.
template <int D, bool FP8, int SCALE, int NT, int STEP, int OCC, bool Q_LDS, bool STREAM>
__global__ __launch_bounds__(64 * kBlockWaves) __attribute__((amdgpu_waves_per_eu(OCC, OCC)))
void pa_block_attention_kernel(const PaBlockArgs a, const BlockCut cut) {
  constexpr int ESZ = FP8 ? 1 : 2;
  constexpr int X = FP8 ? 16 : 8;            // cache elements per 16 bytes
  constexpr int KL = D / (4 * X);            // 16-byte K loads per lane and tile
  constexpr int KM = D / 32;                 // MFMAs per tile of S
  constexpr int DB = D / 16;                 // 16-dim rows of O
  constexpr int NP = STEP / 16;              // pieces of a step, and tiles of S
  constexpr int TPL = STEP / 4;              // tokens of a lane
  constexpr int U = TPL / 8;                 // MFMAs per 16 dims of O and P term
  constexpr int VW = TPL * ESZ / 4;          // V words per lane and 16 dims
  constexpr int OROW = D + 4;                // floats per row of the merge buffer (padded: rows on different banks)
  static_assert(STEP == 64 || STEP == 32, "a lane has a whole piece or half of one");
  __shared__ __attribute__((aligned(16))) float o_lds[kBlockWaves][16][OROW];
  __shared__ float m_lds[kBlockWaves][16], l_lds[kBlockWaves][16];
  u32x4* const q_lds = reinterpret_cast<u32x4*>(&o_lds[0][0][0]);  // (the query operands, until the waves merge)
  static_assert(!Q_LDS || NT * KM * 64 * 16 <= (int)sizeof(o_lds), "the query operands fit where the waves merge");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, kg = lane >> 4;
  const int Hkv = a.num_kv_heads, G = a.group_size;
  const int Ge = a.q_len * G;

  // ---- which (sequence, stretch, head, row group) ---------------------------------------------------------------------
  const uint32_t units = (uint32_t)(Hkv * cut.row_groups);
  uint32_t unit, item;
  if (cut.spread) {
    unit = blockIdx.x % units;
    item = blockIdx.x / units;
  } else {
    // workgroup ids go round the eight XCDs: an item's heads and row groups are consecutive workgroups of one XCD, so the
    // 128-byte lines that hold neighbouring heads' scales, and pages that several row groups read, are fetched once
    const uint32_t slot = blockIdx.x >> 3;
    unit = slot % units;
    item = slot / units * 8u + (blockIdx.x & 7u);
    if (item >= (uint32_t)a.num_seqs * (uint32_t)cut.parts) return;
  }
  const int h = (int)(unit % (uint32_t)Hkv);
  const int row0 = (int)(unit / (uint32_t)Hkv) * 16 * NT;
  const int b = (int)(item % (uint32_t)a.num_seqs);
  const int part = (int)(item / (uint32_t)a.num_seqs);

  int ctx = sload_i32(a.context_lens + b);
  ctx = ctx < 0 ? 0 : (ctx > cut.axis ? cut.axis : ctx);
  const int end_v = virtual_tokens(a, b, h, ctx);
  const int wg_start = part * cut.part;
  if (wg_start >= end_v && cut.parts > 1) return;  // (nobody reads this stretch's partial result)
  const int wg_end = min(wg_start + cut.part, end_v);
  int qb = a.q_lens ? sload_i32(a.q_lens + b) : a.q_len;
  qb = qb < 0 ? 0 : (qb > a.q_len ? a.q_len : qb);
  const int rows_valid = qb * G;

  // logits in the log2 domain: k_factor * (q . k), with the factor's sign moved into q (a maximum is then one of q . k)
  float k_factor = a.softmax_scale * kLog2e, v_factor = 1.f;
  if constexpr (SCALE == kScaleOne) {
    if (a.kv_quant_mode == PA_QUANT_PER_TENSOR) {
      k_factor *= sload_f32(a.key_scale);
      v_factor = sload_f32(a.value_scale);
    }
  }
  const uint32_t flip = k_factor < 0.f ? 0x80008000u : 0u;
  k_factor = fabsf(k_factor);

  // ---- the query rows: FP8, MFMA c = 2 g + m takes head dims 64 g + 16 kg + 8 m .. + 7 (half of the lane's 16-byte
  // piece of K); bf16, 32 c + 8 kg .. + 7 ---------------------------------------------------------------------------------
  bf16x8 q[Q_LDS ? 1 : NT][Q_LDS ? 1 : KM];
  auto query_operand = [&](int n, int c) {
    const int row = row0 + 16 * n + li;
    const int d = FP8 ? 64 * (c >> 1) + 16 * kg + 8 * (c & 1) : 32 * c + 8 * kg;
    u32x4 r = {0, 0, 0, 0};
    if (row < rows_valid) r = load16((const __bf16*)a.query + (int64_t)b * a.stride_q_s + (int64_t)(h * Ge + row) * a.stride_q_h + d) ^ flip;
    return r;
  };
  if constexpr (Q_LDS) {
    for (int i = wave; i < NT * KM; i += kBlockWaves) q_lds[i * 64 + lane] = query_operand(i / KM, i % KM);
    __syncthreads();
  } else {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < KM; ++c) q[n][c] = Bf16x8Bits{.u = query_operand(n, c)}.v;
    }
  }
  auto q_of = [&](int n, int c) {
    if constexpr (Q_LDS)
      return Bf16x8Bits{.u = q_lds[(n * KM + c) * 64 + lane]}.v;
    else
      return q[n][c];
  };
  int limit[NT];  // keys the lane's row sees (causal over the new tokens)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = row0 + 16 * n + li;
    limit[n] = row < rows_valid ? ctx - (qb - 1 - row / G) : 0;
  }
  const int limit_all = ctx - (a.q_len - 1);  // keys that every row sees, at least

  const int log2_bs = 31 - __builtin_clz(a.block_size);
  const int bs_mask = a.block_size - 1;
  const int num_logical = (ctx + bs_mask) >> log2_bs;
  const int* table = a.block_tables + (int64_t)b * a.stride_bt_s;
  const int* list = a.selected_blocks ? a.selected_blocks + (int64_t)b * a.stride_sel_s + (int64_t)h * a.stride_sel_h : nullptr;
  const char* kbase = (const char*)a.key_cache + (int64_t)h * a.stride_k_h * ESZ;
  const char* vbase = (const char*)a.value_cache + (int64_t)h * a.stride_v_h * ESZ;
  const int64_t scale_h = (int64_t)h * a.stride_kvscale_h;

  // One step's pieces: the cache block of each, the token's offset in it and its position in the sequence.  A piece that
  // is not there (behind the stretch, a number outside the sequence, an entry outside the cache) reads block 0 and has a
  // position behind every context.
  struct Pieces {
    int page[NP], off[NP], pos[NP];
  };
  constexpr int kNowhere = 0x7fffff00;
  auto fetch = [&](int tok0) {
    Pieces p;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int t = tok0 + 16 * j;
      const bool in = t < wg_end;
      const int idx = in ? t >> log2_bs : 0;
      int logical = list ? sload_i32(list + idx) : idx;
      bool ok = in && (unsigned)logical < (unsigned)num_logical;
      const int page = sload_i32(table + (ok ? logical : 0));
      ok = ok && (unsigned)page < (unsigned)a.num_blocks;
      p.page[j] = ok ? page : 0;
      p.off[j] = t & bs_mask;
      p.pos[j] = ok ? (logical << log2_bs) + p.off[j] : kNowhere;
    }
    return p;
  };
  // the piece of lane group g, and where in it the group's tokens begin
  auto pick = [](const int (&v)[NP], int g) {
    if constexpr (NP == 4)
      return g == 0 ? v[0] : g == 1 ? v[1] : g == 2 ? v[2] : v[3];
    else
      return g < 2 ? v[0] : v[1];
  };
  auto inside = [](int g) { return NP == 4 ? 0 : 8 * (g & 1); };
  const int sub = li >> 2;  // the lane group whose tokens this lane's K rows are; kg is the one its logits and V are of

  u32x4 kr[NP][KL];
  uint32_t vr[DB][VW];
  f32x4 ks[SCALE == kScaleToken ? NP : 1], vs[SCALE == kScaleToken ? NP : 1];
  float ks1 = 1.f, vs1 = 1.f;
  auto load_k = [&](const Pieces& p) {
    const char* kt = kbase + (int64_t)pick(p.page, sub) * a.stride_k_b * ESZ + (pick(p.off, sub) + inside(sub) + (li & 3)) * 16;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
#pragma unroll
      for (int g = 0; g < KL; ++g) {
        const char* src = kt + (int64_t)(4 * g + kg) * a.stride_k_c * ESZ + 64 * j;
        kr[j][g] = STREAM ? load16_stream(src) : load16(src);
      }
    }
  };
  auto load_v = [&](const Pieces& p) {
    const int off = pick(p.off, kg) + inside(kg);
    const char* vt = vbase + (int64_t)pick(p.page, kg) * a.stride_v_b * ESZ;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int d = 16 * db + li;
      const int64_t e = a.v_transposed ? (int64_t)(off / X) * a.stride_v_2 + d * X + off % X : (int64_t)d * a.stride_v_2 + off;
      const char* src = vt + e * ESZ;
      if constexpr (VW == 2) {
        const u32x2 w = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(src)) : *reinterpret_cast<const u32x2*>(src);
        vr[db][0] = w[0];
        vr[db][1] = w[1];
      } else {
#pragma unroll
        for (int i = 0; i < VW; i += 4) {
          // (bf16, 16 tokens: the second eight are the next tile of a transposed cache)
          const char* s = i == 0 ? src : src + (a.v_transposed ? a.stride_v_2 : 8) * ESZ;
          const u32x4 w = STREAM ? load16_stream(s) : load16(s);
#pragma unroll
          for (int k = 0; k < 4; ++k) vr[db][i + k] = w[k];
        }
      }
    }
  };
  auto load_scales = [&](const Pieces& p) {
    const int64_t so = (int64_t)pick(p.page, kg) * a.stride_kvscale_b + scale_h;
    if constexpr (SCALE == kScaleBlock) {
      ks1 = a.key_scale[so];
      vs1 = a.value_scale[so];
    } else if constexpr (SCALE == kScaleToken) {
      const int off = pick(p.off, kg) + inside(kg);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        ks[j] = *reinterpret_cast<const f32x4*>(a.key_scale + so + off + 4 * j);
        vs[j] = *reinterpret_cast<const f32x4*>(a.value_scale + so + off + 4 * j);
      }
    }
  };
  // eight tokens (FP8: two words, bf16: four) of a head dim as an MFMA operand, times a power of two (FP8)
  auto v_operand = [&](int db, int u, float pow2) {
    if constexpr (FP8) {
      typedef __attribute__((ext_vector_type(2))) __bf16 pair;
      union {
        pair p[4];
        bf16x8 v;
      } r;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        r.p[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vr[db][2 * u + i], pow2, false);
        r.p[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vr[db][2 * u + i], pow2, true);
      }
      return r.v;
    } else {
      return Bf16x8Bits{.u = u32x4{vr[db][4 * u], vr[db][4 * u + 1], vr[db][4 * u + 2], vr[db][4 * u + 3]}}.v;
    }
  };

  // The reference m_run of row li's sums (log2 domain; the same in the row's four lanes) follows the row's maximum only when
  // that is more than kLag above it: probabilities up to 2^kLag cost no precision, and most steps rescale nothing.
  constexpr float kLag = 8.f;
  float m_run[NT], l_run[NT];
  f32x4 acc[NT][DB];           // O^T: head dims 16 db + 4 kg .. + 3 of row li
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m_run[n] = -INFINITY;
    l_run[n] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[n][db] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  constexpr int kStride = kBlockWaves * STEP;
  int tok0 = wg_start + wave * STEP;
  if (tok0 < wg_end) {
    Pieces now = fetch(tok0);
    load_k(now);
    load_scales(now);
    load_v(now);
    Pieces next = fetch(tok0 + kStride);
    for (; tok0 < wg_end; tok0 += kStride) {
      const bool more = tok0 + kStride < wg_end;
      // (the compiler would otherwise read the query operands once, in front of the loop, into registers that are not there)
      if constexpr (Q_LDS) asm volatile("" ::: "memory");
      // ---- S^T = K Q^T ------------------------------------------------------------------------------------------------
      f32x4 s[NT][NP];
#pragma unroll
      for (int j = 0; j < NP; ++j) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < KL; ++g) {
          if constexpr (FP8) {
            const bf16x8 k0 = fp8x8_to_bf16x8(kr[j][g][0], kr[j][g][1]), k1 = fp8x8_to_bf16x8(kr[j][g][2], kr[j][g][3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              s[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, q_of(n, 2 * g), s[n][j], 0, 0, 0);
              s[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, q_of(n, 2 * g + 1), s[n][j], 0, 0, 0);
            }
          } else {
            Bf16x8Bits k0;
            k0.u = kr[j][g];
#pragma unroll
            for (int n = 0; n < NT; ++n) s[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0.v, q_of(n, g), s[n][j], 0, 0, 0);
          }
        }
      }
      // this step's scales; the registers are about to take the next step's
      f32x4 ks_now[SCALE == kScaleToken ? NP : 1], vs_now[SCALE == kScaleToken ? NP : 1];
      float ks1_now = ks1, vs1_now = vs1;
      if constexpr (SCALE == kScaleToken) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          ks_now[j] = ks[j];
          vs_now[j] = vs[j];
        }
      }
      if (more) {
        load_k(next);
        load_scales(next);
      }
      // ---- softmax (s[n][j][r]: token 4 j + r of the lane's) --------------------------------------------------------------
      const int pos = pick(now.pos, kg) + inside(kg);
      bool plain = pos + TPL <= limit_all;
      if constexpr (SCALE == kScaleBlock) plain = plain && !(fminf(ks1_now, vs1_now) < 0.f);  // (a scale below zero turns the order of the logits)
      const bool clean = __all(plain);
      const int live = ctx - pos;  // live tokens of the lane's (may be <= 0 or >= TPL)
      if (!clean) {  // a scale behind the context may be NaN, and 0 * NaN is NaN
        if constexpr (SCALE == kScaleBlock) vs1_now = live > 0 ? vs1_now : 0.f;
        if constexpr (SCALE == kScaleToken) {
#pragma unroll
          for (int j = 0; j < NP; ++j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) vs_now[j][r] = 4 * j + r < live ? vs_now[j][r] : 0.f;
          }
        }
        // bytes behind the context may decode to NaN: those tokens' V is zero
        if (__any(live < TPL)) {
#pragma unroll
          for (int db = 0; db < DB; ++db) {
#pragma unroll
            for (int w = 0; w < VW; ++w) {
              const int n = live - w * (4 / ESZ);  // live tokens from this word on
              vr[db][w] &= n >= 4 / ESZ ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * ESZ * n)) - 1u);
            }
          }
        }
        // the sign of V's scale goes to the codes
        if constexpr (SCALE == kScaleBlock) {
          if (__any(vs1_now < 0.f)) {
            const uint32_t turn = vs1_now < 0.f ? 0x80808080u : 0u;
#pragma unroll
            for (int db = 0; db < DB; ++db) {
#pragma unroll
              for (int w = 0; w < VW; ++w) vr[db][w] ^= turn;
            }
          }
        }
      }
      // The size of V's scale is 2^e v_rest with v_rest in [1, 2): the power is applied when the codes are converted, v_rest as a
      // summand of the probabilities' exponents, which the lane's sum is rid of again (both are exactly nothing for a power of two)
      float v_pow2 = 1.f, v_log2 = 0.f, v_inv = 1.f;
      if constexpr (SCALE == kScaleBlock) {
        const uint32_t bits = __float_as_uint(vs1_now) & 0x7fffffffu;
        const bool normal = (bits & 0x7f800000u) != 0;
        const float v_rest = normal ? __uint_as_float((bits & 0x7fffffu) | 0x3f800000u) : (bits ? __uint_as_float(bits) * 0x1p126f : 1.f);
        v_pow2 = normal || !bits ? __uint_as_float(bits & 0x7f800000u) : 0x1p-126f;
        v_log2 = fast_log2(v_rest);
        v_inv = __builtin_amdgcn_rcpf(v_rest);
      }
      bf16x8 hi[NT][U], lo[NT][U];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float c = SCALE == kScaleBlock ? ks1_now * k_factor : k_factor;
        if (SCALE == kScaleToken || !clean) {
#pragma unroll
          for (int j = 0; j < NP; ++j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float x = s[n][j][r] * c;
              if constexpr (SCALE == kScaleToken) x *= ks_now[j][r];
              s[n][j][r] = clean || pos + 4 * j + r < limit[n] ? x : -INFINITY;  // (a select: bytes behind the context may be NaN)
            }
          }
          c = 1.f;
        }
        float mx = s[n][0][0];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[n][j][r]);
        }
        mx = quad_row_max(mx * c);
        if (__any(!(mx <= m_run[n] + kLag))) {
          const float m_new = fmaxf(m_run[n], mx);
          const float alpha = fast_exp2(m_run[n] - (m_new == -INFINITY ? 0.f : m_new));  // exp2(-inf) = 0 while the row has seen no key
          m_run[n] = m_new;
          l_run[n] *= alpha;
#pragma unroll
          for (int db = 0; db < DB; ++db) acc[n][db] *= alpha;
        }
        const float m_safe = m_run[n] == -INFINITY ? 0.f : m_run[n];
        const float base = v_log2 - m_safe;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          Bf16x8Bits ph, pl;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float p[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = 2 * u + (w >> 1), r = 2 * (w & 1) + e;
              p[e] = fast_exp2(__builtin_fmaf(s[n][j][r], c, base));
              sum += p[e];
              if constexpr (SCALE == kScaleToken) p[e] *= vs_now[j][r];
            }
            ph.u[w] = pack_bf16x2(p[0], p[1]);
            pl.u[w] = pack_bf16x2(p[0] - bf16_bits_to_f32(ph.u[w] & 0xffffu), p[1] - bf16_bits_to_f32(ph.u[w] >> 16));
          }
          hi[n][u] = ph.v;
          lo[n][u] = pl.v;
        }
        l_run[n] += quad_row_sum(sum * v_inv);
      }
      // ---- O^T += V^T P --------------------------------------------------------------------------------------------------
#pragma unroll
      for (int db = 0; db < DB; ++db) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const bf16x8 v = v_operand(db, u, v_pow2);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[n][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, hi[n][u], acc[n][db], 0, 0, 0);
            acc[n][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, lo[n][u], acc[n][db], 0, 0, 0);
          }
        }
      }
      if (more) {
        load_v(next);
        now = next;
        next = fetch(tok0 + 2 * kStride);
      }
    }
  }

  // ---- the waves' results meet in LDS, one tile after the other ------------------------------------------------------------
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (n || Q_LDS) __syncthreads();
#pragma unroll
    for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(&o_lds[wave][li][16 * db + 4 * kg]) = acc[n][db];
    if (kg == 0) {
      m_lds[wave][li] = m_run[n];
      l_lds[wave][li] = l_run[n];
    }
    __syncthreads();
    const int r = threadIdx.x >> 4, c = threadIdx.x & 15;  // row of the tile; its D / 16 head dims
    const int row = row0 + 16 * n + r;
    if (row < Ge) {
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kBlockWaves; ++w) M = fmaxf(M, m_lds[w][r]);
      const float M_safe = M == -INFINITY ? 0.f : M;
      float L = 0.f, o[DB] = {};
#pragma unroll
      for (int w = 0; w < kBlockWaves; ++w) {
        const float f = fast_exp2(m_lds[w][r] - M_safe);
        L += f * l_lds[w][r];
#pragma unroll
        for (int i = 0; i < DB; i += 4) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(&o_lds[w][r][c * DB + i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i + e] += f * v[e];
        }
      }
      if (cut.parts > 1) {
        const int64_t slot = (((int64_t)b * Hkv + h) * cut.parts + part) * Ge + row;
        float* po = (float*)a.workspace + slot * D + c * DB;
#pragma unroll
        for (int i = 0; i < DB; i += 4) *reinterpret_cast<f32x4*>(po + i) = f32x4{o[i], o[i + 1], o[i + 2], o[i + 3]} * v_factor;
        if (c == 0) {
          float* pm = (float*)a.workspace + (int64_t)a.num_seqs * Hkv * cut.parts * Ge * D + slot * 2;
          pm[0] = M;
          pm[1] = L;
        }
      } else {
        const bool ok = row < rows_valid && L != 0.f;  // (a NaN sum is a result)
        const float inv = ok ? v_factor / L : 0.f;
        __bf16* out = (__bf16*)a.output + (int64_t)b * a.stride_out_s + (int64_t)(h * Ge + row) * a.stride_out_h + c * DB;
#pragma unroll
        for (int i = 0; i < DB; i += 4) {
          u32x2 w;
          w[0] = ok ? pack_bf16x2(o[i] * inv, o[i + 1] * inv) : 0u;
          w[1] = ok ? pack_bf16x2(o[i + 2] * inv, o[i + 3] * inv) : 0u;
          *reinterpret_cast<u32x2*>(out + i) = w;
        }
        if (a.lse && c == 0) a.lse[(int64_t)b * a.stride_lse_s + h * Ge + row] = ok ? (M + fast_log2(L)) * (1.f / kLog2e) : -INFINITY;
      }
    }
  }
}

// Merges the stretches of a cut axis: one workgroup per (sequence, kv head, row); D / 4 lanes take a partial result, the
// workgroup 1024 / D of them at a time.
template <int D>
__global__ __launch_bounds__(256) void pa_block_merge_kernel(const PaBlockArgs a, const BlockCut cut) {
  constexpr int LANES = D / 4, GROUPS = 256 / LANES;
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) float o_lds[GROUPS][D];
  __shared__ float l_lds[GROUPS];
  const int tid = threadIdx.x;
  const int Ge = a.q_len * a.group_size;
  const int row = (int)(blockIdx.x % (unsigned)Ge);
  const unsigned bh = blockIdx.x / (unsigned)Ge;
  const int h = (int)(bh % (unsigned)a.num_kv_heads), b = (int)(bh / (unsigned)a.num_kv_heads);
  int ctx = sload_i32(a.context_lens + b);
  ctx = ctx < 0 ? 0 : (ctx > cut.axis ? cut.axis : ctx);
  int qb = a.q_lens ? sload_i32(a.q_lens + b) : a.q_len;
  qb = qb > a.q_len ? a.q_len : qb;
  const int n = row < qb * a.group_size ? (virtual_tokens(a, b, h, ctx) + cut.part - 1) / cut.part : 0;
  const int64_t slot0 = (int64_t)bh * cut.parts * Ge + row;
  const float* po = (const float*)a.workspace + slot0 * D;
  const float* pm = (const float*)a.workspace + (int64_t)a.num_seqs * a.num_kv_heads * cut.parts * Ge * D + slot0 * 2;
  float M = -INFINITY;
  for (int p = tid; p < n; p += 256) M = fmaxf(M, pm[(int64_t)p * Ge * 2]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
  if ((tid & 63) == 0) red[tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float M_safe = M == -INFINITY ? 0.f : M;
  const int g = tid / LANES, c = tid % LANES;
  float L = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = g; p < n; p += GROUPS) {
    const float f = fast_exp2(pm[(int64_t)p * Ge * 2] - M_safe);
    L += f * pm[(int64_t)p * Ge * 2 + 1];
    o += *reinterpret_cast<const f32x4*>(po + (int64_t)p * Ge * D + 4 * c) * f;
  }
  *reinterpret_cast<f32x4*>(&o_lds[g][4 * c]) = o;
  if (c == 0) l_lds[g] = L;
  __syncthreads();
  if (tid < LANES) {
    L = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      L += l_lds[i];
      o += *reinterpret_cast<const f32x4*>(&o_lds[i][4 * c]);
    }
    const bool ok = L != 0.f;
    const float inv = ok ? 1.f / L : 0.f;
    u32x2 w;
    w[0] = ok ? pack_bf16x2(o[0] * inv, o[1] * inv) : 0u;
    w[1] = ok ? pack_bf16x2(o[2] * inv, o[3] * inv) : 0u;
    *reinterpret_cast<u32x2*>((__bf16*)a.output + (int64_t)b * a.stride_out_s + (int64_t)(h * Ge + row) * a.stride_out_h + 4 * c) = w;
    if (a.lse && c == 0) a.lse[(int64_t)b * a.stride_lse_s + h * Ge + row] = ok ? (M + fast_log2(L)) * (1.f / kLog2e) : -INFINITY;
  }
}

// The same for a few stretches: a wave per row, no barriers.
constexpr int kFewParts = 16;
template <int D>
__global__ __launch_bounds__(256) void pa_block_merge_few_kernel(const PaBlockArgs a, const BlockCut cut) {
  constexpr int LANES = D / 4, GROUPS = 64 / LANES;
  const int lane = threadIdx.x & 63;
  const int Ge = a.q_len * a.group_size;
  const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= (int64_t)a.num_seqs * a.num_kv_heads * Ge) return;
  const int row = (int)(r % Ge), bh = (int)(r / Ge);
  const int h = bh % a.num_kv_heads, b = bh / a.num_kv_heads;
  int ctx = sload_i32(a.context_lens + b);
  ctx = ctx < 0 ? 0 : (ctx > cut.axis ? cut.axis : ctx);
  int qb = a.q_lens ? sload_i32(a.q_lens + b) : a.q_len;
  qb = qb > a.q_len ? a.q_len : qb;
  const int n = row < qb * a.group_size ? (virtual_tokens(a, b, h, ctx) + cut.part - 1) / cut.part : 0;
  const int64_t slot0 = (int64_t)bh * cut.parts * Ge + row;
  const float* po = (const float*)a.workspace + slot0 * D;
  const float* pm = (const float*)a.workspace + (int64_t)a.num_seqs * a.num_kv_heads * cut.parts * Ge * D + slot0 * 2;
  // lane p < n holds stretch p's maximum and sum
  const f32x2 ml = lane < n ? *reinterpret_cast<const f32x2*>(pm + (int64_t)lane * Ge * 2) : f32x2{-INFINITY, 0.f};
  const int g = lane / LANES, c = lane % LANES;
  f32x4 v[kFewParts / GROUPS];
#pragma unroll
  for (int i = 0; i < kFewParts / GROUPS; ++i) {
    const int p = i * GROUPS + g;
    v[i] = p < n ? *reinterpret_cast<const f32x4*>(po + (int64_t)p * Ge * D + 4 * c) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  float M = ml[0];
#pragma unroll
  for (int o = 1; o < kFewParts; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
  M = __shfl(M, 0);
  const float f = fast_exp2(ml[0] - (M == -INFINITY ? 0.f : M));
  float L = lane < n ? f * ml[1] : 0.f;
#pragma unroll
  for (int o = 1; o < kFewParts; o <<= 1) L += __shfl_xor(L, o);
  L = __shfl(L, 0);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kFewParts / GROUPS; ++i) {
    const float w = __shfl(f, i * GROUPS + g);
    if (i * GROUPS + g < n) o += v[i] * w;
  }
#pragma unroll
  for (int d = LANES; d < 64; d <<= 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], d);
  }
  if (g == 0) {
    const bool ok = L != 0.f;
    const float inv = ok ? 1.f / L : 0.f;
    u32x2 w;
    w[0] = ok ? pack_bf16x2(o[0] * inv, o[1] * inv) : 0u;
    w[1] = ok ? pack_bf16x2(o[2] * inv, o[3] * inv) : 0u;
    *reinterpret_cast<u32x2*>((__bf16*)a.output + (int64_t)b * a.stride_out_s + (int64_t)(h * Ge + row) * a.stride_out_h + 4 * c) = w;
    if (a.lse && c == 0) a.lse[(int64_t)b * a.stride_lse_s + h * Ge + row] = ok ? (M + fast_log2(L)) * (1.f / kLog2e) : -INFINITY;
  }
}

int check_attention(const PaBlockArgs* a) {
  if (int rc = check_block_sizes(a)) return rc;
  if (int rc = check_block_rows(a)) return rc;
  if (int rc = check_block_cache(a, true)) return rc;
  if (!a->output || !a->query) return PA_ERR_NULL_POINTER;
  if (!block_aligned16(a->query) || a->stride_q_s % 8 || a->stride_q_h % 8) return PA_ERR_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(a->output) & 7) || a->stride_out_s % 4 || a->stride_out_h % 4) return PA_ERR_BAD_SHAPE;
  if (a->selected_blocks && (a->num_selected <= 0 || (int64_t)a->num_selected * a->block_size > 0x40000000LL)) return PA_ERR_BAD_SHAPE;
  if (!a->selected_blocks && a->selected_counts) return PA_ERR_NULL_POINTER;
  return PA_OK;
}

// 16-row query tiles of a workgroup: as many as the call has, up to what the registers hold
int row_tiles(const PaBlockArgs& a) {
  const int tiles = (a.group_size * a.q_len + 15) / 16;
  if (tiles == 1 || (a.head_size == 256 && a.kv_dtype == PA_DTYPE_BF16)) return 1;
  return 2;
}

BlockCut choose_cut(const PaBlockArgs& a) {
  BlockCut c;
  c.axis = block_axis(a);
  const int nt = row_tiles(a);
  c.row_groups = (a.group_size * a.q_len + 16 * nt - 1) / (16 * nt);
  const int64_t axis = a.selected_blocks ? (int64_t)a.num_selected * a.block_size : c.axis;
  const int64_t units = (int64_t)a.num_seqs * a.num_kv_heads * c.row_groups;
  int64_t parts = (512 + units - 1) / units;             // two workgroups for each of 256 CUs
  if (parts * 4096 < axis) parts = (axis + 4096 - 1) / 4096;  // a ragged batch's longest sequence is no tail of its own
  if (parts > (axis + 255) / 256) parts = (axis + 255) / 256;
  if (parts < 1) parts = 1;
  const int64_t per = (axis + parts - 1) / parts;
  c.part = (int)((per + 255) / 256 * 256);
  if (c.part < 256) c.part = 256;
  c.parts = (int)((axis + c.part - 1) / c.part);
  if (c.parts < 1) c.parts = 1;
  c.spread = (int64_t)a.num_seqs * c.parts < 64;  // fewer items leave XCDs without work when each takes whole items
  return c;
}

int64_t workspace_of(const PaBlockArgs& a, const BlockCut& c) {
  if (c.parts <= 1) return 0;
  return (int64_t)a.num_seqs * a.num_kv_heads * c.parts * a.group_size * a.q_len * (a.head_size + 2) * 4;
}

template <int D, bool FP8, int SCALE, int NT>
int launch_tile(const PaBlockArgs& a, const BlockCut& c, dim3 grid, hipStream_t s) {
  // what a wave has in flight, the query operands and the accumulators share 256 registers (two waves per SIMD), or 512
  constexpr int OCC = D == 256 && (!FP8 || NT > 1) ? 1 : 2;
  constexpr int STEP = D == 256 || !FP8 || (D == 128 && SCALE == kScaleToken && NT > 1) ? 32 : 64;
  constexpr bool Q_LDS = NT > 1 || D == 256;
  // (16-token FP8 blocks that one workgroup reads whole and nobody else reads: loads that do not stay in L2)
  if constexpr (FP8 && NT == 1)
    if (a.block_size == 16 && c.row_groups == 1)
      return pa_launch(pa_block_attention_kernel<D, FP8, SCALE, NT, STEP, OCC, Q_LDS, true>, grid, dim3(64 * kBlockWaves), 0, s, a, c);
  return pa_launch(pa_block_attention_kernel<D, FP8, SCALE, NT, STEP, OCC, Q_LDS, false>, grid, dim3(64 * kBlockWaves), 0, s, a, c);
}

template <int D, bool FP8, int SCALE>
int launch_tiles(const PaBlockArgs& a, const BlockCut& c, dim3 grid, hipStream_t s) {
  if constexpr (D < 256 || FP8)
    if (row_tiles(a) == 2) return launch_tile<D, FP8, SCALE, 2>(a, c, grid, s);
  return launch_tile<D, FP8, SCALE, 1>(a, c, grid, s);
}

template <int D>
int launch_scale(const PaBlockArgs& a, const BlockCut& c, dim3 grid, hipStream_t s) {
  if (a.kv_dtype == PA_DTYPE_BF16) return launch_tiles<D, false, kScaleOne>(a, c, grid, s);
  if (a.kv_quant_mode == PA_QUANT_PER_TOKEN) return launch_tiles<D, true, kScaleToken>(a, c, grid, s);
  if (a.kv_quant_mode == PA_QUANT_PER_BLOCK) return launch_tiles<D, true, kScaleBlock>(a, c, grid, s);
  return launch_tiles<D, true, kScaleOne>(a, c, grid, s);
}

}  // namespace

extern "C" {

uint32_t pa_block_args_size(void) { return (uint32_t)sizeof(PaBlockArgs); }

int64_t pa_block_attention_workspace_bytes(const PaBlockArgs* a) {
  if (int rc = check_attention(a)) return rc;
  return workspace_of(*a, choose_cut(*a));
}

int pa_block_attention(const PaBlockArgs* a, void* hip_stream) {
  if (int rc = check_attention(a)) return rc;
  const BlockCut c = choose_cut(*a);
  const int64_t need = workspace_of(*a, c);
  if (need > 0) {
    if (!a->workspace) return PA_ERR_NULL_POINTER;
    if (a->workspace_bytes < need || !block_aligned16(a->workspace)) return PA_ERR_SCRATCH_TOO_SMALL;
  }
  const int64_t items = (int64_t)a->num_seqs * c.parts, units = (int64_t)a->num_kv_heads * c.row_groups;
  const int64_t wgs = c.spread ? items * units : (items + 7) / 8 * 8 * units;
  const int64_t rows = (int64_t)a->num_seqs * a->num_kv_heads * a->group_size * a->q_len;
  if (wgs > 0x7fffffffLL || rows > 0x7fffffffLL) return PA_ERR_BAD_SHAPE;
  hipStream_t s = reinterpret_cast<hipStream_t>(hip_stream);
  const dim3 grid((unsigned)wgs);
  const int rc = a->head_size == 64    ? launch_scale<64>(*a, c, grid, s)
                 : a->head_size == 128 ? launch_scale<128>(*a, c, grid, s)
                                       : launch_scale<256>(*a, c, grid, s);
  if (rc || c.parts == 1) return rc;
  if (c.parts <= kFewParts) {
    const dim3 few((unsigned)((rows + 3) / 4));
    return a->head_size == 64    ? pa_launch(pa_block_merge_few_kernel<64>, few, dim3(256), 0, s, *a, c)
           : a->head_size == 128 ? pa_launch(pa_block_merge_few_kernel<128>, few, dim3(256), 0, s, *a, c)
                                 : pa_launch(pa_block_merge_few_kernel<256>, few, dim3(256), 0, s, *a, c);
  }
  const dim3 mgrid((unsigned)rows);
  return a->head_size == 64    ? pa_launch(pa_block_merge_kernel<64>, mgrid, dim3(256), 0, s, *a, c)
         : a->head_size == 128 ? pa_launch(pa_block_merge_kernel<128>, mgrid, dim3(256), 0, s, *a, c)
                               : pa_launch(pa_block_merge_kernel<256>, mgrid, dim3(256), 0, s, *a, c);
}

}  // extern "C"
