// Shared by the block-granular operators (pa_block_attention.hip, pa_block_select.hip): what their arguments have to
// satisfy before anything is launched.
#ifndef PA_BLOCK_H_
#define PA_BLOCK_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/pa_decode.h"
#include "pa_launch.h"

namespace {

inline bool block_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// sizes that every entry point reads; 0 or an error code
inline int check_block_sizes(const PaBlockArgs* a) {
  if (!a) return PA_ERR_NULL_POINTER;
  if (a->struct_size != sizeof(PaBlockArgs)) return PA_ERR_BAD_STRUCT;
  if (!a->context_lens || !a->block_tables) return PA_ERR_NULL_POINTER;
  if (a->num_seqs <= 0 || a->num_kv_heads <= 0 || a->num_blocks <= 0 || a->table_width <= 0 || a->max_context_len < 0)
    return PA_ERR_BAD_SHAPE;
  if (a->reserved0 != 0 || a->reserved1 != 0) return PA_ERR_BAD_SHAPE;
  if (a->head_size != 64 && a->head_size != 128 && a->head_size != 256) return PA_ERR_UNSUPPORTED;
  if (a->block_size != 16 && a->block_size != 64 && a->block_size != 1024) return PA_ERR_UNSUPPORTED;
  if (a->stride_bt_s < 0) return PA_ERR_BAD_SHAPE;
  // token positions and counts of (sequence, head, block) are 32-bit in the kernels
  if ((int64_t)a->table_width * a->block_size > 0x40000000LL || a->max_context_len > 0x40000000) return PA_ERR_BAD_SHAPE;
  if ((int64_t)a->num_seqs * a->num_kv_heads > 0x7ffffff) return PA_ERR_BAD_SHAPE;
  return PA_OK;
}

// the query rows of a call
inline int check_block_rows(const PaBlockArgs* a) {
  if (a->group_size <= 0 || a->q_len <= 0) return PA_ERR_BAD_SHAPE;
  if ((int64_t)a->group_size * a->q_len > 64) return PA_ERR_UNSUPPORTED;
  return PA_OK;
}

inline int check_block_cache(const PaBlockArgs* a, bool value) {
  if (!a->key_cache || (value && !a->value_cache)) return PA_ERR_NULL_POINTER;
  if (a->kv_dtype != PA_DTYPE_BF16 && a->kv_dtype != PA_DTYPE_FP8_E4M3FN) return PA_ERR_UNSUPPORTED;
  if (a->kv_quant_mode < PA_QUANT_NONE || a->kv_quant_mode > PA_QUANT_PER_BLOCK) return PA_ERR_UNSUPPORTED;
  if (a->kv_dtype == PA_DTYPE_BF16 && a->kv_quant_mode != PA_QUANT_NONE) return PA_ERR_UNSUPPORTED;
  if (a->kv_quant_mode != PA_QUANT_NONE && (!a->key_scale || (value && !a->value_scale))) return PA_ERR_NULL_POINTER;
  if (a->kv_quant_mode == PA_QUANT_PER_TOKEN &&
      (a->stride_kvscale_b % 4 || a->stride_kvscale_h % 4 || !block_aligned16(a->key_scale) || (value && !block_aligned16(a->value_scale))))
    return PA_ERR_BAD_SHAPE;
  if (a->v_transposed != 0 && a->v_transposed != 1) return PA_ERR_BAD_SHAPE;
  // the kernels move 16 bytes at a time
  const int x = a->kv_dtype == PA_DTYPE_FP8_E4M3FN ? 16 : 8;
  if (!block_aligned16(a->key_cache) || a->stride_k_b % x || a->stride_k_h % x || a->stride_k_c % x) return PA_ERR_BAD_SHAPE;
  if (value && (!block_aligned16(a->value_cache) || a->stride_v_b % x || a->stride_v_h % x || a->stride_v_2 % x)) return PA_ERR_BAD_SHAPE;
  return PA_OK;
}

// tokens of the longest context that the call can reach
inline int block_axis(const PaBlockArgs& a) {
  const int64_t reach = (int64_t)a.table_width * a.block_size;
  return (int)(a.max_context_len < reach ? a.max_context_len : reach);
}

}  // namespace

#endif  // PA_BLOCK_H_
