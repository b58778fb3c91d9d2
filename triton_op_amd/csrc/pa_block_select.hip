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
// One wave per (sequence, visited block, kv head); lane l owns head dims l, l + 64, ...
template <int D, bool FP8>
__global__ __launch_bounds__(64) void pa_block_bounds_kernel(const PaBlockArgs a, const int axis, const int visits) {
  const int lane = threadIdx.x;
  const int h = (int)(blockIdx.x % (unsigned)a.num_kv_heads);
  const int item = (int)(blockIdx.x / (unsigned)a.num_kv_heads);
  const int b = item / visits;
  const int ctx = block_context(a, b, axis);
  const int bs = a.block_size;
  const int first = a.new_tokens > 0 ? (ctx > a.new_tokens ? ctx - a.new_tokens : 0) / bs : 0;
  const int at = first + item % visits;
  if (at * bs >= ctx) return;
  const int page = a.block_tables[(int64_t)b * a.stride_bt_s + at];
  if ((unsigned)page >= (unsigned)a.num_blocks) return;
  const int live = ctx - at * bs < bs ? ctx - at * bs : bs;
  constexpr int X = FP8 ? 16 : 8;
  const char* kp = (const char*)a.key_cache + ((int64_t)page * a.stride_k_b + (int64_t)h * a.stride_k_h) * (FP8 ? 1 : 2);
  const float* sp = a.key_scale + (int64_t)page * a.stride_kvscale_b + (int64_t)h * a.stride_kvscale_h;
  __bf16* out = (__bf16*)a.bounds + (int64_t)page * a.stride_bounds_b + (int64_t)h * a.stride_bounds_h;
  for (int d = lane; d < D; d += 64) {
    float lo = INFINITY, hi = -INFINITY;
    for (int t = 0; t < live; ++t) {
      const int64_t e = (int64_t)(d / X) * a.stride_k_c + t * X + d % X;
      float x;
      if constexpr (FP8)
        x = __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)kp)[e], 0);
      else
        x = bf16_bits_to_f32(((const uint16_t*)kp)[e]);
      if (a.kv_quant_mode == PA_QUANT_PER_TENSOR) x *= a.key_scale[0];
      if (a.kv_quant_mode == PA_QUANT_PER_TOKEN) x *= sp[t];
      if (a.kv_quant_mode == PA_QUANT_PER_BLOCK) x *= sp[0];
      if (x < lo) lo = x;
      if (x > hi) hi = x;
    }
    out[d] = (__bf16)lo;
    out[D + d] = (__bf16)hi;
  }
}

// ---- scores ------------------------------------------------------------------------------------------------------------
// a score as a key whose unsigned order is the scores' order; forced blocks have the largest key, which no score has
constexpr unsigned long long kForcedKey = ~0ull;
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (s != s) s = -INFINITY;  // no row had a number
  s = s + 0.0;                // -0 and +0 are equal scores
  const unsigned long long u = (unsigned long long)__double_as_longlong(s);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// One wave per (sequence, kv head, block): the key of every block into the workspace [B, Hkv, axis blocks].
template <int D>
__global__ __launch_bounds__(64) void pa_block_score_kernel(const PaBlockArgs a, const int axis, const int axis_blocks) {
  const int lane = threadIdx.x;
  const int h = (int)(blockIdx.x % (unsigned)a.num_kv_heads);
  const unsigned item = blockIdx.x / (unsigned)a.num_kv_heads;
  const int b = (int)(item / (unsigned)axis_blocks), at = (int)(item % (unsigned)axis_blocks);
  const int ctx = block_context(a, b, axis);
  const int nb = (ctx + a.block_size - 1) / a.block_size;
  if (at >= nb) return;
  unsigned long long* key = (unsigned long long*)a.workspace + ((int64_t)b * a.num_kv_heads + h) * axis_blocks + at;
  if (at < a.first_blocks || at >= nb - a.recent_blocks) {
    if (lane == 0) *key = kForcedKey;
    return;
  }
  const int page = a.block_tables[(int64_t)b * a.stride_bt_s + at];
  double best = -INFINITY;
  if ((unsigned)page < (unsigned)a.num_blocks) {
    const __bf16* box = (const __bf16*)a.bounds + (int64_t)page * a.stride_bounds_b + (int64_t)h * a.stride_bounds_h;
    int qb = a.q_lens ? a.q_lens[b] : a.q_len;
    qb = qb > a.q_len ? a.q_len : qb;
    const int Ge = a.q_len * a.group_size;
    for (int row = 0; row < qb * a.group_size; ++row) {
      const __bf16* q = (const __bf16*)a.query + (int64_t)b * a.stride_q_s + (int64_t)(h * Ge + row) * a.stride_q_h;
      double s = 0.0;
      for (int d = lane; d < D; d += 64) {
        const double x = (double)(float)q[d];
        s += (x > 0.0 ? x : 0.0) * (double)(float)box[D + d] + (x < 0.0 ? x : 0.0) * (double)(float)box[d];
      }
      for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
      if (s == INFINITY) s = 0x1.fffffffffffffp1023;
      if (s > best) best = s;  // (a NaN is passed over)
    }
  }
  if (lane == 0) *key = score_key(best);
}

// ---- selection -----------------------------------------------------------------------------------------------------------
// One workgroup per (sequence, kv head): the K-th largest key by eight passes over its bytes, then the blocks above it
// and the first of the blocks that equal it, in ascending order.
constexpr int kSelectThreads = 1024;
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
  for (int w = 0; w < kSelectThreads / 64; ++w) {
    const int v = wave_sums[w];
    before += w < wave ? v : 0;
    total += v;
  }
  return before + s - x;
}

__global__ __launch_bounds__(kSelectThreads) void pa_block_select_kernel(const PaBlockArgs a, const int axis, const int axis_blocks) {
  __shared__ int hist[256];
  __shared__ int wave_sums[kSelectThreads / 64];
  __shared__ int digit, above;
  const int tid = threadIdx.x;
  const int h = (int)(blockIdx.x % (unsigned)a.num_kv_heads), b = (int)(blockIdx.x / (unsigned)a.num_kv_heads);
  const int ctx = block_context(a, b, axis);
  const int nb = (ctx + a.block_size - 1) / a.block_size;
  const int K = a.num_selected;
  int32_t* out = a.selected_blocks + (int64_t)b * a.stride_sel_s + (int64_t)h * a.stride_sel_h;
  const int count = nb < K ? nb : K;
  if (tid == 0) a.selected_counts[(int64_t)b * a.stride_cnt_s + h] = count;
  for (int i = count + tid; i < K; i += kSelectThreads) out[i] = -1;
  if (nb <= K) {
    for (int i = tid; i < nb; i += kSelectThreads) out[i] = i;
    return;
  }
  const unsigned long long* key = (const unsigned long long*)a.workspace + ((int64_t)b * a.num_kv_heads + h) * axis_blocks;
  unsigned long long prefix = 0;
  int want = K;  // of the keys that share the digits fixed so far, how many are still to be taken
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < nb; i += kSelectThreads) {
      const unsigned long long k = key[i];
      if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int sum = 0, v = 255;
      for (; v > 0; --v) {
        if (sum + hist[v] >= want) break;
        sum += hist[v];
      }
      digit = v;
      above = sum;
    }
    __syncthreads();
    prefix |= (unsigned long long)digit << shift;
    want -= above;
  }
  // keys above the threshold, and the first `want` that equal it
  int done = 0, equal_before = 0;
  for (int i0 = 0; i0 < nb; i0 += kSelectThreads) {
    const int i = i0 + tid;
    const unsigned long long k = i < nb ? key[i] : 0;
    const bool eq = i < nb && k == prefix;
    int total;
    const int rank = equal_before + workgroup_scan(eq, wave_sums, total);
    equal_before += total;
    const bool take = i < nb && (k > prefix || (eq && rank < want));
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
  const int64_t grid = (int64_t)a->num_seqs * visits * a->num_kv_heads;
  if (grid > 0x7fffffffLL) return PA_ERR_BAD_SHAPE;
  const dim3 g((unsigned)grid), t(64);
  const bool fp8 = a->kv_dtype == PA_DTYPE_FP8_E4M3FN;
  switch (a->head_size) {
    case 64:
      return fp8 ? pa_launch(pa_block_bounds_kernel<64, true>, g, t, 0, stream, *a, axis, visits)
                 : pa_launch(pa_block_bounds_kernel<64, false>, g, t, 0, stream, *a, axis, visits);
    case 128:
      return fp8 ? pa_launch(pa_block_bounds_kernel<128, true>, g, t, 0, stream, *a, axis, visits)
                 : pa_launch(pa_block_bounds_kernel<128, false>, g, t, 0, stream, *a, axis, visits);
    default:
      return fp8 ? pa_launch(pa_block_bounds_kernel<256, true>, g, t, 0, stream, *a, axis, visits)
                 : pa_launch(pa_block_bounds_kernel<256, false>, g, t, 0, stream, *a, axis, visits);
  }
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
  const int64_t grid = (int64_t)a->num_seqs * blocks * a->num_kv_heads;
  if (grid > 0x7fffffffLL) return PA_ERR_BAD_SHAPE;
  const dim3 g((unsigned)grid), t(64);
  const int rc = a->head_size == 64    ? pa_launch(pa_block_score_kernel<64>, g, t, 0, stream, *a, axis, blocks)
                 : a->head_size == 128 ? pa_launch(pa_block_score_kernel<128>, g, t, 0, stream, *a, axis, blocks)
                                       : pa_launch(pa_block_score_kernel<256>, g, t, 0, stream, *a, axis, blocks);
  if (rc) return rc;
  return pa_launch(pa_block_select_kernel, dim3((unsigned)(a->num_seqs * a->num_kv_heads)), dim3(kSelectThreads), 0, stream, *a, axis, blocks);
}

}  // extern "C"
