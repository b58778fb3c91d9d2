// KV-cache write into an FP8 cache with one scale per (block, kv head): pa_kv_cache_write_block_scaled.
//
//   s_new = max(s_old, 2^ceil(log2(amax / 448)))      amax over the new rows that stay in the block
//   code  = e4m3(code * (s_old / s_new))              codes that were there, when the scale grew (s_old > 0)
//   code  = e4m3(x / s_new)                           new rows
//
// A block's scale depends on all of the call's rows that land in it, so a block must have ONE owner.  The owner is the
// workgroup of the first token of the call that lies in the block: it finds the block's other tokens by reading the
// whole slot mapping (64 KiB for 8192 tokens, from L2), and no workspace, no sort and no second launch is needed.
// Per slot the latest token is kept (an LDS maximum of token numbers), so the bytes do not depend on timing.
// From there on a wave owns a (block, kv head) and needs no barrier: it goes through the block's 16-slot segments that
// change, 16 bytes of a row per lane.  K leaves as 8-byte halves of (chunk, token) cells, V is turned in LDS so that a
// head dim's 16 tokens are one 16-byte store, new codes among the old ones.  Every byte is written at most once.
// Bound by the chain of latencies slot -> slot mapping -> rows -> store: 64 tokens x 8 heads 8 us, 8192 tokens (50 MB) 22 us = 2.3
// TB/s in blocks of 16; the read of the slot mapping grows with its square (65536 tokens: 260 us).
// Larger blocks have fewer owners, and a wave goes through its block's segments one after the other, twice: 8192 tokens take 46 us in
// blocks of 64 and 0.52 ms in blocks of 1024 (8 workgroups at work).  A scale that grows rewrites the whole block, also slots
// that hold nothing yet: a step of 64 tokens whose scales all grow takes 8, 20 and 250 us in blocks of 16, 64 and 1024.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/pa_decode.h"
#include "pa_launch.h"

namespace {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

constexpr int kThreads = 256;
constexpr int kMaxBlockSize = 1024;

// four values to four e4m3 codes: saturating, a NaN stays a NaN
__device__ __forceinline__ float clamp_code(float x) { return x != x ? x : __builtin_amdgcn_fmed3f(x, -448.f, 448.f); }
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_code(a), clamp_code(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(clamp_code(c), clamp_code(d), w, true);
}
// e4m3(code * ratio) of four codes; 0 < ratio <= 1
__device__ __forceinline__ uint32_t rescale_codes(uint32_t w, float ratio) {
  return to_codes(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * ratio,
                  __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * ratio);
}

// the smallest power of two s >= 2^-126 with amax <= 448 s, for a bf16 amax given by its bits (finite, sign cleared).
// 448 = 1.75 * 2^8, so the exponent is that of amax minus 8, plus one if its significand is above 1.75.
__device__ __forceinline__ float scale_for(uint32_t amax_bits16) {
  const uint32_t u = amax_bits16 << 16;
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(e < 1 ? 1 : e) << 23);
}

// largest finite magnitude (bits) of the two bf16 values of a word
__device__ __forceinline__ uint32_t finite_max2(uint32_t m, uint32_t w) {
  const uint32_t lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
  m = lo < 0x7f80u && lo > m ? lo : m;
  return hi < 0x7f80u && hi > m ? hi : m;
}

// 8 consecutive bf16 values of a row
template <bool ALIGNED>
__device__ __forceinline__ u32x4 load_row8(const uint16_t* p) {
  if constexpr (ALIGNED) {
    return *reinterpret_cast<const u32x4*>(p);
  } else {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return r;
  }
}

// Eight codes of x / s, given 1 / s in 64 bits.  For a power of two s the 32-bit product is the quotient.  For any other s
// the 64-bit product, rounded to 32 bits, is the correctly rounded 32-bit quotient: x has 8 significant bits and s 24, so x / s
// is never closer than 2^-49 to a midpoint of 32-bit numbers (that midpoint times s has 25 significant bits or more, x has 8),
// and the product is off by 2^-51 at most.
__device__ __forceinline__ u32x2 quantize_row8(u32x4 x, double inv, bool pow2) {
  u32x2 out;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t p = x[2 * w + (e >> 1)];
      v[e] = __uint_as_float(e & 1 ? p & 0xffff0000u : p << 16);
    }
    if (pow2) {
      const float r = (float)inv;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= r;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (float)((double)v[e] * inv);
    }
    out[w] = to_codes(v[0], v[1], v[2], v[3]);
  }
  return out;
}

// 4x4 transpose of bytes: word i holds byte j of row i, afterwards byte i of column j
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// One (block, kv head), by one wave.  owner: the block's slots' tokens (LDS); segs: the segments that get a token.
template <int D, bool ALIGNED>
__device__ __forceinline__ void write_block_head(const PaKvWriteArgs& a, const long long block, const int h, const int bs, const int* owner,
                                                 const unsigned long long segs, uint8_t (*turn)[D], const int lane) {
  constexpr int P = D / 8;         // lanes of a row, 8 head dims each
  constexpr int R = 16 * P / 64;   // loads per lane for 16 rows
  constexpr int DL = D / 4;        // lanes that hold four head dims of V each
  const uint16_t* key = (const uint16_t*)a.key + (int64_t)h * a.stride_k_h + lane % P * 8;
  const uint16_t* value = (const uint16_t*)a.value + (int64_t)h * a.stride_v_h + lane % P * 8;
  uint8_t* kc = (uint8_t*)a.key_cache + block * a.stride_kc_b + (int64_t)h * a.stride_kc_h;
  uint8_t* vc = (uint8_t*)a.value_cache + block * a.stride_vc_b + (int64_t)h * a.stride_vc_h;
  const int64_t so = block * a.stride_scale_b + (int64_t)h * a.stride_scale_h;
  const float old_k = a.key_scale[so], old_v = a.value_scale[so];

  u32x4 kr[R], vr[R], was[4];
  auto token_of = [&](int seg, int j) { return owner[16 * seg + lane / P + 64 / P * j]; };
  auto load_rows = [&](int seg) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int tok = token_of(seg, j);
      kr[j] = vr[j] = u32x4{0, 0, 0, 0};
      if (tok >= 0) {
        kr[j] = load_row8<ALIGNED>(key + (int64_t)tok * a.stride_k_t);
        vr[j] = load_row8<ALIGNED>(value + (int64_t)tok * a.stride_v_t);
      }
    }
  };
  // lane's four head dims 4 lane + i of V: 16 tokens each
  auto v_row = [&](int seg, int i) {
    const int d = 4 * lane + i;
    return reinterpret_cast<u32x4*>(vc + (a.v_transposed ? ((int64_t)seg * D + d) * 16 : (int64_t)d * bs + 16 * seg));
  };
  auto member_mask = [&](int seg) {
    return (uint32_t)__builtin_amdgcn_ballot_w64(owner[16 * seg + (lane & 15)] >= 0) & 0xffffu;
  };
  auto load_was = [&](int seg, uint32_t members) {
    if (members != 0xffffu && lane < DL) {
#pragma unroll
      for (int i = 0; i < 4; ++i) was[i] = *v_row(seg, i);
    }
  };

  // ---- amax of the new rows: the last segment's rows stay in registers ---------------------------------------------------
  uint32_t mk = 0, mv = 0;
  int held = -1;
  for (unsigned long long left = segs; left; left &= left - 1) {
    held = __builtin_ctzll(left);
    load_rows(held);
    if (!(left & (left - 1))) load_was(held, member_mask(held));
#pragma unroll
    for (int j = 0; j < R; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        mk = finite_max2(mk, kr[j][e]);
        mv = finite_max2(mv, vr[j][e]);
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t ok = __shfl_xor(mk, o), ov = __shfl_xor(mv, o);
    mk = ok > mk ? ok : mk;
    mv = ov > mv ? ov : mv;
  }
  const float new_k = fmaxf(old_k, scale_for(mk)), new_v = fmaxf(old_v, scale_for(mv));
  const bool grow_k = old_k > 0.f && new_k > old_k, grow_v = old_v > 0.f && new_v > old_v;
  const float ratio_k = grow_k ? __fdiv_rn(old_k, new_k) : 1.f, ratio_v = grow_v ? __fdiv_rn(old_v, new_v) : 1.f;
  auto is_pow2 = [](float s) { return (__float_as_uint(s) & 0x7fffffu) == 0 && s >= 0x1p-126f && s <= 0x1p126f; };
  const bool pow2_k = is_pow2(new_k), pow2_v = is_pow2(new_v);
  const double inv_k = 1.0 / (double)new_k, inv_v = 1.0 / (double)new_v;
  if (lane == 0) {
    a.key_scale[so] = new_k;
    a.value_scale[so] = new_v;
  }

  // ---- the segments that change, the one in registers first -----------------------------------------------------------------
  const unsigned long long all = bs == 1024 ? ~0ull : (1ull << (bs >> 4)) - 1;
  unsigned long long left = grow_k || grow_v ? all : segs;
  for (int seg = held; left;) {
    const uint32_t members = member_mask(seg);
    if (seg != held) {
      load_rows(seg);
      if (members || grow_v) load_was(seg, members);
    }
    // K: the lane's 8 head dims of a token are half of a 16-byte (chunk, token) cell
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int slot = 16 * seg + lane / P + 64 / P * j, c = lane % P;
      if (owner[slot] >= 0)
        *reinterpret_cast<u32x2*>(kc + ((int64_t)(c >> 1) * bs + slot) * 16 + 8 * (c & 1)) = quantize_row8(kr[j], inv_k, pow2_k);
    }
    if (grow_k) {
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const int cell = lane + 64 * i, slot = 16 * seg + (cell & 15);
        if (owner[slot] >= 0) continue;
        u32x4* p = reinterpret_cast<u32x4*>(kc + ((int64_t)(cell >> 4) * bs + slot) * 16);
        u32x4 w = *p;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = rescale_codes(w[e], ratio_k);
        *p = w;
      }
    }
    // V: codes into LDS as rows, out of it as columns
    if (members || grow_v) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        *reinterpret_cast<u32x2*>(&turn[lane / P + 64 / P * j][lane % P * 8]) = quantize_row8(vr[j], inv_v, pow2_v);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      if (lane < DL) {
        u32x4 out[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // tokens 4 e .. 4 e + 3
          uint32_t w[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) w[t] = *reinterpret_cast<const uint32_t*>(&turn[4 * e + t][4 * lane]);
          transpose4(w);
          const uint32_t m = members >> (4 * e) & 15u;  // bytes that are new
          const uint32_t take = (m & 1 ? 0xffu : 0u) | (m & 2 ? 0xff00u : 0u) | (m & 4 ? 0xff0000u : 0u) | (m & 8 ? 0xff000000u : 0u);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t o = 0;
            if (members != 0xffffu) o = grow_v ? rescale_codes(was[i][e], ratio_v) : was[i][e];
            out[i][e] = (w[i] & take) | (o & ~take);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) *v_row(seg, i) = out[i];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    left &= ~(1ull << seg);
    seg = left ? __builtin_ctzll(left) : 0;
  }
}

// grid: (windows of `window` tokens) x (groups of `heads` kv heads).  ALIGNED: the rows can be read 16 bytes at a time.
template <int D, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void kv_cache_write_block_scaled_kernel(const PaKvWriteArgs a, const long long num_slots,
                                                                               const int bs_shift, const int window, const int turn_bits,
                                                                               const int heads) {
  __shared__ int owner[kMaxBlockSize];     // per slot of the block: the latest token of the call, -1 without one
  __shared__ unsigned long long segments;  // bit i: 16-slot segment i gets a token
  __shared__ int earlier;
  __shared__ __attribute__((aligned(16))) uint8_t turn[kThreads / 64][16][D];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bs = 1 << bs_shift;
  const int num_tokens = (int)a.num_tokens;
  const int head_groups = (a.num_kv_heads + heads - 1) / heads;
  // Workgroups are handed out in id order, round the XCDs and round the shader engines of each, and one that has to wait for
  // its engine holds up the next.  In a prompt every fourth window owns a block (16-token blocks): in plain order these
  // would all be one engine's (measured: 4 times the time).  Bits of the id in reverse order make them neighbours.
  const unsigned unit = blockIdx.x / (unsigned)head_groups, group = (1u << turn_bits) - 1;
  const unsigned turned = turn_bits ? __builtin_bitreverse32(unit & group) >> (32 - turn_bits) : 0;
  const long long t0 = (long long)((unit & ~group) | turned) * window;
  if (t0 >= num_tokens) return;
  const int h0 = (int)(blockIdx.x % (unsigned)head_groups) * heads;
  const int h1 = h0 + heads < a.num_kv_heads ? h0 + heads : a.num_kv_heads;
  const int t_end = (int)(t0 + window < num_tokens ? t0 + window : num_tokens);

  auto block_of = [&](long long slot) -> long long { return slot < 0 || slot >= num_slots ? -1 : slot >> bs_shift; };
  // the tokens of the window that begin a run in their block (most tokens of a prompt do not)
  const int mine = (int)t0 + lane;
  bool begins = false;
  if (lane < window && mine < t_end) {
    const long long block = block_of(a.slot_mapping[mine]);
    begins = block >= 0 && (mine == 0 || block_of(a.slot_mapping[mine - 1]) != block);
  }
  for (uint64_t todo = __builtin_amdgcn_ballot_w64(begins); todo; todo &= todo - 1) {
    const int t = (int)t0 + __builtin_ctzll(todo);
    const long long block = a.slot_mapping[t] >> bs_shift;
    __syncthreads();  // the previous block's lists are done with
    for (int i = tid; i < bs; i += kThreads) owner[i] = -1;
    if (tid == 0) {
      earlier = 0;
      segments = 0;
    }
    __syncthreads();
    // (eight slots of a thread are asked for at a time: one by one this would be a chain of L2 latencies)
    for (int i0 = tid; i0 < num_tokens; i0 += 8 * kThreads) {
      long long slot[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * kThreads;
        slot[u] = i < num_tokens ? a.slot_mapping[i] : -1;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (block_of(slot[u]) != block) continue;
        const int i = i0 + u * kThreads, off = (int)(slot[u] & (bs - 1));
        if (i < t) {
          earlier = 1;
        } else {
          atomicMax(&owner[off], i);
          atomicOr(&segments, 1ull << (off >> 4));
        }
      }
    }
    __syncthreads();
    if (earlier) continue;  // another workgroup (or an earlier turn of this one) owns the block
    for (int h = h0 + wave; h < h1; h += kThreads / 64) write_block_head<D, ALIGNED>(a, block, h, bs, owner, segments, turn[wave], lane);
  }
}

}  // namespace

extern "C" int pa_kv_cache_write_block_scaled(const PaKvWriteArgs* a, int64_t num_blocks, void* hip_stream) {
  if (!a) return PA_ERR_NULL_POINTER;
  if (a->struct_size != sizeof(PaKvWriteArgs)) return PA_ERR_BAD_STRUCT;
  if (a->num_tokens == 0) return PA_OK;  // (an empty tensor has no address)
  if (!a->key || !a->value || !a->slot_mapping || !a->key_cache || !a->value_cache || !a->key_scale || !a->value_scale)
    return PA_ERR_NULL_POINTER;
  if (a->num_tokens < 0 || a->num_tokens > 0x3fffffff || a->num_kv_heads <= 0 || num_blocks <= 0) return PA_ERR_BAD_SHAPE;
  if (a->cache_dtype != PA_DTYPE_FP8_E4M3FN || a->kv_quant_mode != PA_QUANT_PER_BLOCK) return PA_ERR_UNSUPPORTED;
  if (a->head_size != 64 && a->head_size != 128 && a->head_size != 256) return PA_ERR_UNSUPPORTED;
  if (a->block_size != 16 && a->block_size != 64 && a->block_size != 1024) return PA_ERR_UNSUPPORTED;
  if (a->v_transposed != 0 && a->v_transposed != 1) return PA_ERR_BAD_SHAPE;
  const uintptr_t caches = reinterpret_cast<uintptr_t>(a->key_cache) | reinterpret_cast<uintptr_t>(a->value_cache);
  if ((caches & 15) || a->stride_kc_b % 16 || a->stride_kc_h % 16 || a->stride_vc_b % 16 || a->stride_vc_h % 16) return PA_ERR_BAD_SHAPE;
  const uintptr_t rows = reinterpret_cast<uintptr_t>(a->key) | reinterpret_cast<uintptr_t>(a->value);
  const bool aligned = (rows & 15) == 0 && a->stride_k_t % 8 == 0 && a->stride_k_h % 8 == 0 && a->stride_v_t % 8 == 0 && a->stride_v_h % 8 == 0;
  // (Both cuts are for blocks of 16 tokens; larger blocks have the same.)
  // A few tokens (decode): one workgroup per (token, four kv heads).  Many (prompts): most tokens own no block, so a
  // workgroup looks at four of them, and walks all kv heads so that the slot mapping is read once per block (8192 tokens, 8
  // heads: 28 us with windows of 16, where one workgroup in a prompt has two blocks, 23 with 4).
  const bool many = a->num_tokens > 1024;
  const int window = many ? 4 : 1, heads = many ? a->num_kv_heads : kThreads / 64;
  const int64_t windows = (a->num_tokens + window - 1) / window;
  int turn_bits = 0;
  while (turn_bits < 10 && (1 << turn_bits) < windows) ++turn_bits;
  const int64_t grid = ((windows + (1 << turn_bits) - 1) >> turn_bits << turn_bits) * ((a->num_kv_heads + heads - 1) / heads);
  if (grid > 0x7fffffffLL) return PA_ERR_BAD_SHAPE;
  const int shift = __builtin_ctz((unsigned)a->block_size);
  const long long num_slots = num_blocks << shift;
  hipStream_t stream = reinterpret_cast<hipStream_t>(hip_stream);
  const dim3 g((unsigned)grid), b(kThreads);
#define PA_WRITE(D)                                                                                                               \
  (aligned ? pa_launch(kv_cache_write_block_scaled_kernel<D, true>, g, b, 0, stream, *a, num_slots, shift, window, turn_bits, heads)         \
           : pa_launch(kv_cache_write_block_scaled_kernel<D, false>, g, b, 0, stream, *a, num_slots, shift, window, turn_bits, heads))
  return a->head_size == 64 ? PA_WRITE(64) : a->head_size == 128 ? PA_WRITE(128) : PA_WRITE(256);
#undef PA_WRITE
}
