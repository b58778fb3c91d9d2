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
// Every byte of the block is written at most once: K in 16-byte (chunk, token) cells, V in 16-byte rows of 16 tokens that
// mix new codes with old ones.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/pa_decode.h"
#include "pa_launch.h"

namespace {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

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
__device__ __forceinline__ float bf16_value(uint32_t bits16) { return __uint_as_float(bits16 << 16); }

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

// grid: (windows of `window` tokens) x (groups of `heads` kv heads).  ALIGNED: the rows can be read 16 bytes at a time.
template <int D, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void kv_cache_write_block_scaled_kernel(const PaKvWriteArgs a, const long long num_slots,
                                                                               const int bs_shift, const int window, const int heads) {
  __shared__ int owner[kMaxBlockSize];             // per slot of the block: the latest token of the call, -1 without one
  __shared__ uint16_t member[kMaxBlockSize];       // the slots that get a token, in any order
  __shared__ int count, earlier;
  __shared__ unsigned long long segments;          // bit i: 16-slot segment i gets a token
  __shared__ uint32_t amax[2];
  const int tid = threadIdx.x;
  const int bs = 1 << bs_shift, nseg = bs >> 4;
  const int num_tokens = (int)a.num_tokens;
  const int head_groups = (a.num_kv_heads + heads - 1) / heads;
  const int h0 = (int)(blockIdx.x % (unsigned)head_groups) * heads;
  const int h1 = h0 + heads < a.num_kv_heads ? h0 + heads : a.num_kv_heads;
  const long long t0 = (long long)(blockIdx.x / (unsigned)head_groups) * window;
  const long long t_end = t0 + window < num_tokens ? t0 + window : num_tokens;

  auto block_of = [&](long long t) -> long long {
    const long long slot = a.slot_mapping[t];
    return slot < 0 || slot >= num_slots ? -1 : slot >> bs_shift;
  };
  for (int t = (int)t0; t < t_end; ++t) {
    const long long block = block_of(t);
    if (block < 0 || (t > 0 && block_of(t - 1) == block)) continue;  // (most tokens of a prompt: their run began earlier)
    __syncthreads();  // the previous block's lists are done with
    for (int i = tid; i < bs; i += kThreads) owner[i] = -1;
    if (tid == 0) {
      count = earlier = 0;
      segments = 0;
    }
    __syncthreads();
    for (int i = tid; i < num_tokens; i += kThreads) {
      const long long slot = a.slot_mapping[i];
      if (slot < 0 || slot >= num_slots || slot >> bs_shift != block) continue;
      if (i < t)
        earlier = 1;
      else
        atomicMax(&owner[slot & (bs - 1)], i);
    }
    __syncthreads();
    if (earlier) continue;  // another workgroup (or an earlier turn of this one) owns the block
    for (int i = tid; i < bs; i += kThreads) {
      if (owner[i] < 0) continue;
      member[atomicAdd(&count, 1)] = (uint16_t)i;
      atomicOr(&segments, 1ull << (i >> 4));
    }
    __syncthreads();
    const int n = count;
    const unsigned long long segs = segments;

    for (int h = h0; h < h1; ++h) {
      const uint16_t* key = (const uint16_t*)a.key + (int64_t)h * a.stride_k_h;
      const uint16_t* value = (const uint16_t*)a.value + (int64_t)h * a.stride_v_h;
      // ---- amax of the new rows -----------------------------------------------------------------------------------
      if (tid < 2) amax[tid] = 0;
      __syncthreads();
      uint32_t mk = 0, mv = 0;
      for (int i = tid; i < n * (D / 8); i += kThreads) {
        const int64_t tok = owner[member[i / (D / 8)]];
        const int d = i % (D / 8) * 8;
        const u32x4 k8 = load_row8<ALIGNED>(key + tok * a.stride_k_t + d), v8 = load_row8<ALIGNED>(value + tok * a.stride_v_t + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          mk = finite_max2(mk, k8[e]);
          mv = finite_max2(mv, v8[e]);
        }
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const uint32_t ok = __shfl_xor(mk, o), ov = __shfl_xor(mv, o);
        mk = ok > mk ? ok : mk;
        mv = ov > mv ? ov : mv;
      }
      if ((tid & 63) == 0) {
        atomicMax(&amax[0], mk);
        atomicMax(&amax[1], mv);
      }
      // every thread reads the old scales before the barrier that lets thread 0 write the new ones
      const int64_t so = block * a.stride_scale_b + (int64_t)h * a.stride_scale_h;
      const float old_k = a.key_scale[so], old_v = a.value_scale[so];
      __syncthreads();
      const float new_k = fmaxf(old_k, scale_for(amax[0])), new_v = fmaxf(old_v, scale_for(amax[1]));
      const bool grow_k = old_k > 0.f && new_k > old_k, grow_v = old_v > 0.f && new_v > old_v;
      const float ratio_k = grow_k ? __fdiv_rn(old_k, new_k) : 1.f, ratio_v = grow_v ? __fdiv_rn(old_v, new_v) : 1.f;
      if (tid == 0) {
        a.key_scale[so] = new_k;
        a.value_scale[so] = new_v;
      }
      // ---- K: 16-byte cells (16 head dims of a token) --------------------------------------------------------------------
      uint8_t* kc = (uint8_t*)a.key_cache + block * a.stride_kc_b + (int64_t)h * a.stride_kc_h;
      for (int i = tid; i < n * (D / 16); i += kThreads) {
        const int off = member[i / (D / 16)], c = i % (D / 16);
        const uint16_t* row = key + (int64_t)owner[off] * a.stride_k_t + 16 * c;
        const u32x4 x0 = load_row8<ALIGNED>(row), x1 = load_row8<ALIGNED>(row + 8);
        u32x4 out;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t p = w < 2 ? x0[2 * w] : x1[2 * w - 4], q = w < 2 ? x0[2 * w + 1] : x1[2 * w - 3];
          out[w] = to_codes(__fdiv_rn(bf16_value(p & 0xffffu), new_k), __fdiv_rn(bf16_value(p >> 16), new_k),
                            __fdiv_rn(bf16_value(q & 0xffffu), new_k), __fdiv_rn(bf16_value(q >> 16), new_k));
        }
        *reinterpret_cast<u32x4*>(kc + ((int64_t)c * bs + off) * 16) = out;
      }
      if (grow_k) {
        for (int i = tid; i < bs * (D / 16); i += kThreads) {
          if (owner[i & (bs - 1)] >= 0) continue;
          u32x4* p = reinterpret_cast<u32x4*>(kc + (int64_t)i * 16);
          u32x4 w = *p;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = rescale_codes(w[e], ratio_k);
          *p = w;
        }
      }
      // ---- V: 16 tokens of a head dim, new codes among the old ones ---------------------------------------------------------
      uint8_t* vc = (uint8_t*)a.value_cache + block * a.stride_vc_b + (int64_t)h * a.stride_vc_h;
      constexpr int kSegs = kThreads / D;  // segments the workgroup takes at a time, D threads each
      const int d = tid % D;
      for (int seg = tid / D; seg < nseg; seg += kSegs) {
        if (!grow_v && !((segs >> seg) & 1)) continue;
        u32x4* p = reinterpret_cast<u32x4*>(vc + (a.v_transposed ? ((int64_t)seg * D + d) * 16 : (int64_t)d * bs + 16 * seg));
        u32x4 w = *p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (grow_v) w[e] = rescale_codes(w[e], ratio_v);
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int tok = owner[16 * seg + 4 * e + b];
            if (tok < 0) continue;
            const float x = bf16_value(value[(int64_t)tok * a.stride_v_t + d]);
            const uint32_t code = to_codes(__fdiv_rn(x, new_v), 0.f, 0.f, 0.f) & 0xffu;
            w[e] = (w[e] & ~(0xffu << (8 * b))) | (code << (8 * b));
          }
        }
        *p = w;
      }
      __syncthreads();  // amax is free for the next head
    }
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
  // a few tokens (decode): one workgroup per (token, kv head).  Many (prompts): most tokens own no block, so a
  // workgroup looks at 16 of them, and walks all kv heads so that the slot mapping is read once per block.
  const bool many = a->num_tokens > 1024;
  const int window = many ? 16 : 1, heads = many ? a->num_kv_heads : 1;
  const int64_t grid = ((a->num_tokens + window - 1) / window) * ((a->num_kv_heads + heads - 1) / heads);
  if (grid > 0x7fffffffLL) return PA_ERR_BAD_SHAPE;
  const int shift = __builtin_ctz((unsigned)a->block_size);
  const long long num_slots = num_blocks << shift;
  hipStream_t stream = reinterpret_cast<hipStream_t>(hip_stream);
  const dim3 g((unsigned)grid), b(kThreads);
#define PA_WRITE(D)                                                                                                               \
  (aligned ? pa_launch(kv_cache_write_block_scaled_kernel<D, true>, g, b, 0, stream, *a, num_slots, shift, window, heads)         \
           : pa_launch(kv_cache_write_block_scaled_kernel<D, false>, g, b, 0, stream, *a, num_slots, shift, window, heads))
  return a->head_size == 64 ? PA_WRITE(64) : a->head_size == 128 ? PA_WRITE(128) : PA_WRITE(256);
#undef PA_WRITE
}
