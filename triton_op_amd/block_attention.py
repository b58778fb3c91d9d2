"""Decode attention at the granularity of cache blocks, and the sparse decode built on it.

* `paged_block_attention` reads a paged cache whose FP8 codes have one scale per (block, kv head)
  ([num_blocks, num_kv_heads, 1, 1]; also per token, per tensor, or none, and bf16 caches), over all blocks of a
  sequence or over the blocks a list names for each (sequence, kv head), and can return the log-sum-exp of every row.
* `key_block_bounds` keeps the smallest and largest key of every block, per kv head and head dimension.
* `select_blocks` picks, for each (sequence, kv head), the blocks whose bounds allow the largest q . k.

A sparse decode step is `kv_cache_write`, `key_block_bounds(..., new_tokens=q)`, `select_blocks`,
`paged_block_attention(..., selected_blocks=...)`.  Query rows, cache layouts, block tables and lengths are those of
`paged_attention_decode`.  All four run HIP kernels of libpa_decode.so on torch's current stream of the tensors' device,
read nothing back to the host and can be captured into a graph; there is no torch implementation behind them.
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional, Tuple

import torch

from . import _cabi
from ._cabi import PaBlockArgs
from .kv_cache import FP8_DTYPE

_SUPPORTED_BLOCK_SIZES = (16, 64, 1024)
_SUPPORTED_HEAD_SIZES = (64, 128, 256)


def _on(dev: torch.device):
    """The context in which a launch on `dev` is made: nothing when it is the current device already."""
    if dev.index is None or dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _strides(t: torch.Tensor) -> Tuple[int, ...]:
    """Strides with 0 for a dimension of size 1, whose stride means nothing."""
    return tuple(st if n > 1 else 0 for n, st in zip(t.shape, t.stride()))


def _same_device(dev, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the call on {dev}")


def _check_sequences(a: PaBlockArgs, sequence_lengths, block_tables, max_sequence_length) -> None:
    if sequence_lengths.dtype != torch.int32 or block_tables.dtype != torch.int32:
        raise ValueError("sequence_lengths and block_tables must be int32")
    if block_tables.dim() != 2 or sequence_lengths.numel() != block_tables.shape[0] or block_tables.shape[1] < 1:
        raise ValueError("sequence_lengths / block_tables do not have one row per sequence")
    if not sequence_lengths.is_contiguous() or (block_tables.shape[1] > 1 and block_tables.stride(1) != 1):
        raise ValueError("sequence_lengths and the rows of block_tables must be contiguous")
    a.context_lens, a.block_tables = sequence_lengths.data_ptr(), block_tables.data_ptr()
    a.num_seqs, a.table_width = block_tables.shape
    a.stride_bt_s = block_tables.stride(0)
    a.max_context_len = max(0, int(max_sequence_length))


def _check_query(a: PaBlockArgs, query, query_sequence_length, num_kv_heads, query_lens) -> None:
    if query.dim() != 3:
        raise ValueError(f"Expected 3D query tensor, but got shape {tuple(query.shape)}")
    if query.dtype != torch.bfloat16:
        raise ValueError(f"query tensor only supports dtype bfloat16, but got {query.dtype}")
    q_len = int(query_sequence_length)
    num_seqs, rows, head_size = query.shape
    if q_len < 1 or rows == 0 or rows % (q_len * num_kv_heads):
        raise ValueError(f"query.shape[1]={rows} is not num_kv_heads*query_sequence_length*group ({num_kv_heads}*{q_len}*G)")
    if rows // num_kv_heads > 64:
        raise ValueError(f"{rows // num_kv_heads} query rows per kv head exceed the maximum of 64")
    if num_seqs != a.num_seqs:
        raise ValueError("sequence_lengths / block_tables do not have one row per sequence")
    if head_size not in _SUPPORTED_HEAD_SIZES:
        raise ValueError(f"head_size == {head_size} is not supported (64, 128 or 256)")
    if query.stride(2) != 1 or query.stride(0) % 8 or query.stride(1) % 8 or query.data_ptr() % 16:
        raise ValueError("query rows must be dense and 16-byte aligned")
    if query_lens is not None:
        if query_lens.dtype != torch.int32 or query_lens.numel() != num_seqs or not query_lens.is_contiguous():
            raise ValueError("query_lens must be contiguous int32 [num_seqs]")
        a.q_lens = query_lens.data_ptr()
    a.query = query.data_ptr()
    a.q_len, a.group_size, a.head_size = q_len, rows // (q_len * num_kv_heads), head_size
    a.stride_q_s, a.stride_q_h = query.stride(0), query.stride(1)


def _check_block_size(block_size: int) -> None:
    if block_size not in _SUPPORTED_BLOCK_SIZES:
        raise ValueError(f"kv_block_size == {block_size} not in {list(_SUPPORTED_BLOCK_SIZES)}")


def _check_key_cache(a: PaBlockArgs, key_cache) -> None:
    if key_cache.dim() != 5:
        raise ValueError(f"Expected 5D key_cache tensor, but got shape {tuple(key_cache.shape)}")
    if key_cache.dtype == FP8_DTYPE:
        a.kv_dtype, x = _cabi.PA_DTYPE_FP8_E4M3FN, 16
    elif key_cache.dtype == torch.bfloat16:
        a.kv_dtype, x = _cabi.PA_DTYPE_BF16, 8
    else:
        raise ValueError(f"key_cache tensor only supports dtype bfloat16 or float8_e4m3fn, but got {key_cache.dtype}")
    blocks, heads, chunks, bs, inner = key_cache.shape
    _check_block_size(bs)
    if inner != x or chunks * x not in _SUPPORTED_HEAD_SIZES or blocks < 1 or heads < 1:
        raise ValueError(f"key_cache shape {tuple(key_cache.shape)} is not [blocks, kv_heads, head_size//{x}, bs, {x}] "
                         "with a head size of 64, 128 or 256")
    st = key_cache.stride()
    if st[4] != 1 or st[3] != x or st[0] % x or st[1] % x or st[2] % x or key_cache.data_ptr() % 16:
        raise ValueError("the innermost dimensions of key_cache must be dense and 16-byte aligned")
    a.key_cache = key_cache.data_ptr()
    a.num_blocks, a.num_kv_heads, a.block_size, a.head_size = blocks, heads, bs, chunks * x
    a.stride_k_b, a.stride_k_h, a.stride_k_c = st[0], st[1], st[2]


def _check_scales(a: PaBlockArgs, key_scale, value_scale, both: bool) -> None:
    a.kv_quant_mode = _cabi.PA_QUANT_NONE
    if both and (key_scale is None) != (value_scale is None):
        raise ValueError("key_scale and value_scale must be given together")
    if key_scale is None:
        return
    if a.kv_dtype != _cabi.PA_DTYPE_FP8_E4M3FN:
        raise ValueError("scales need an FP8 cache")
    for name, s in (("key_scale", key_scale), ("value_scale", value_scale)):
        if s is not None and s.dtype != torch.float32:
            raise ValueError(f"{name} tensor only support dtype == torch.float32")
    if both and (key_scale.shape != value_scale.shape or _strides(key_scale) != _strides(value_scale)):
        raise ValueError("key and value scales must have the same shape and strides")
    shape = tuple(key_scale.shape)
    if shape == ():
        a.kv_quant_mode = _cabi.PA_QUANT_PER_TENSOR
    elif shape == (a.num_blocks, a.num_kv_heads, 1, 1):
        a.kv_quant_mode = _cabi.PA_QUANT_PER_BLOCK
    elif shape == (a.num_blocks, a.num_kv_heads, a.block_size, 1):
        if key_scale.stride(2) != 1 or key_scale.stride(0) % 4 or key_scale.stride(1) % 4 or key_scale.data_ptr() % 16 or \
                (both and value_scale.data_ptr() % 16):
            raise ValueError("per-token scales must be dense over tokens and 16-byte aligned")
        a.kv_quant_mode = _cabi.PA_QUANT_PER_TOKEN
    else:
        raise ValueError(f"Expected scales of shape [], [{a.num_blocks}, {a.num_kv_heads}, 1, 1] or "
                         f"[{a.num_blocks}, {a.num_kv_heads}, {a.block_size}, 1], got {shape}")
    if shape:
        a.stride_kvscale_b, a.stride_kvscale_h = key_scale.stride(0), key_scale.stride(1)
    a.key_scale = key_scale.data_ptr()
    if both:
        a.value_scale = value_scale.data_ptr()


def _check_bounds(a: PaBlockArgs, bounds) -> None:
    if bounds.dtype != torch.bfloat16 or bounds.dim() != 4 or bounds.shape[2] != 2:
        raise ValueError("bounds must be bfloat16 [num_blocks, num_kv_heads, 2, head_size]")
    st = bounds.stride()
    if st[3] != 1 or st[2] != bounds.shape[3] or st[0] % 8 or st[1] % 8 or bounds.data_ptr() % 16:
        raise ValueError("the two bounds of a (block, head) must be dense and 16-byte aligned")
    a.bounds = bounds.data_ptr()
    a.stride_bounds_b, a.stride_bounds_h = st[0], st[1]


class BlockAttentionPlan:
    """A validated call: the filled C struct plus the tensors it points to (kept alive).  `run()` enqueues it on a
    stream; it allocates nothing and can be replayed, and captured.  Plans that may overlap on the GPU need a
    workspace each (a plan made without one has its own)."""

    def __init__(self, args: PaBlockArgs, keep, output):
        self.args, self._keep, self.output = args, keep, output
        self._lib = _cabi.load_library()

    def run(self, stream: Optional[int] = None) -> None:
        if not self.args.num_seqs:
            return
        dev = self.output.device
        with _on(dev):
            if stream is None:
                stream = torch.cuda.current_stream(dev).cuda_stream
            _cabi.check(self._lib.pa_block_attention(C.byref(self.args), C.c_void_p(stream)), "pa_block_attention")


def plan_block_attention(
    output: torch.Tensor,            # [num_seqs, num_kv_heads * query_sequence_length * group, head_size] bf16
    query: torch.Tensor,             # the same shape, bf16
    key_cache: torch.Tensor,         # [num_blocks, num_kv_heads, head_size/x, block_size, x]
    value_cache: torch.Tensor,       # [num_blocks, num_kv_heads, head_size, block_size] or transposed 5-D
    sequence_lengths: torch.Tensor,  # [num_seqs] int32
    block_tables: torch.Tensor,      # [num_seqs, max_num_blocks_per_seq] int32
    softmax_scale: float,
    query_sequence_length: int,
    max_sequence_length: int,
    key_scale: Optional[torch.Tensor] = None,    # [num_blocks, num_kv_heads, 1, 1], [.., block_size, 1] or 0-dim
    value_scale: Optional[torch.Tensor] = None,
    *,
    selected_blocks: Optional[torch.Tensor] = None,  # [num_seqs, num_kv_heads, k] int32, logical block numbers
    selected_counts: Optional[torch.Tensor] = None,  # [num_seqs, num_kv_heads] int32
    query_lens: Optional[torch.Tensor] = None,       # [num_seqs] int32
    lse: Optional[torch.Tensor] = None,              # [num_seqs, rows] f32, written
    workspace: Optional[torch.Tensor] = None,        # uint8
) -> BlockAttentionPlan:
    a = PaBlockArgs()
    a.struct_size = C.sizeof(PaBlockArgs)
    dev = output.device
    _same_device(dev, query=query, key_cache=key_cache, value_cache=value_cache, sequence_lengths=sequence_lengths,
                 block_tables=block_tables, key_scale=key_scale, value_scale=value_scale, selected_blocks=selected_blocks,
                 selected_counts=selected_counts, query_lens=query_lens, lse=lse, workspace=workspace)
    _check_sequences(a, sequence_lengths, block_tables, max_sequence_length)
    _check_key_cache(a, key_cache)
    head_size, bs, heads = a.head_size, a.block_size, a.num_kv_heads
    _check_query(a, query, query_sequence_length, heads, query_lens)
    if a.head_size != head_size:
        raise ValueError(f"query has head size {a.head_size}, key_cache {head_size}")
    if output.shape != query.shape or output.dtype != torch.bfloat16:
        raise ValueError(f"output must be bfloat16 {tuple(query.shape)}, got {output.dtype} {tuple(output.shape)}")
    if output.stride(2) != 1 or output.stride(0) % 4 or output.stride(1) % 4 or output.data_ptr() % 8:
        raise ValueError("output rows must be dense and 8-byte aligned")
    # ---- value cache ---------------------------------------------------------------------------------------------------
    x = 16 // key_cache.element_size()
    if value_cache.dtype != key_cache.dtype:
        raise ValueError(f"value_cache dtype {value_cache.dtype} differs from key_cache dtype {key_cache.dtype}")
    a.v_transposed = int(value_cache.dim() == 5)
    inner = (bs // x, head_size, x) if a.v_transposed else (head_size, bs)
    if tuple(value_cache.shape) != (a.num_blocks, heads) + inner:
        raise ValueError(f"value_cache shape {tuple(value_cache.shape)} is not [blocks, kv_heads, D, bs] or, transposed, "
                         f"[blocks, kv_heads, bs/{x}, D, {x}] of the key cache")
    st = value_cache.stride()
    if st[-1] != 1 or (a.v_transposed and st[3] != x) or any(s % x for s in st[:3]) or value_cache.data_ptr() % 16:
        raise ValueError("the innermost dimensions of value_cache must be dense and 16-byte aligned")
    a.value_cache = value_cache.data_ptr()
    a.stride_v_b, a.stride_v_h, a.stride_v_2 = st[0], st[1], st[2]
    _check_scales(a, key_scale, value_scale, True)
    # ---- the list ----------------------------------------------------------------------------------------------------------
    if selected_blocks is not None:
        if selected_blocks.dtype != torch.int32 or selected_blocks.dim() != 3 or \
                tuple(selected_blocks.shape[:2]) != (a.num_seqs, heads) or selected_blocks.shape[2] < 1:
            raise ValueError(f"selected_blocks must be int32 [{a.num_seqs}, {heads}, k]")
        if selected_blocks.shape[2] > 1 and selected_blocks.stride(2) != 1:
            raise ValueError("selected_blocks must be contiguous in its last dimension")
        a.selected_blocks, a.num_selected = selected_blocks.data_ptr(), selected_blocks.shape[2]
        a.stride_sel_s, a.stride_sel_h = selected_blocks.stride(0), selected_blocks.stride(1)
    if selected_counts is not None:
        if selected_blocks is None:
            raise ValueError("selected_counts needs selected_blocks")
        if selected_counts.dtype != torch.int32 or tuple(selected_counts.shape) != (a.num_seqs, heads) or \
                (heads > 1 and selected_counts.stride(1) != 1):
            raise ValueError(f"selected_counts must be int32 [{a.num_seqs}, {heads}], dense over the heads")
        a.selected_counts, a.stride_cnt_s = selected_counts.data_ptr(), selected_counts.stride(0)
    if lse is not None:
        if lse.dtype != torch.float32 or tuple(lse.shape) != tuple(query.shape[:2]) or lse.stride(1) != 1:
            raise ValueError(f"lse must be float32 {tuple(query.shape[:2])}, dense over the rows")
        a.lse, a.stride_lse_s = lse.data_ptr(), lse.stride(0)
    a.output = output.data_ptr()
    a.stride_out_s, a.stride_out_h = output.stride(0), output.stride(1)
    a.softmax_scale = float(softmax_scale)
    if not output.is_cuda:
        raise ValueError("paged_block_attention runs on the GPU only (there is no CPU path); got a CPU tensor")
    keep = (output, query, key_cache, value_cache, sequence_lengths, block_tables, key_scale, value_scale,
            selected_blocks, selected_counts, query_lens, lse)
    if a.num_seqs:
        need = _workspace_bytes("pa_block_attention_workspace_bytes", a)
        keep += (_give_workspace(a, workspace, need, dev),)
    return BlockAttentionPlan(a, keep, output)


def _workspace_bytes(name: str, a: PaBlockArgs) -> int:
    need = getattr(_cabi.load_library(), name)(C.byref(a))
    if need < 0:
        _cabi.check(int(need), name)
    return need


def _give_workspace(a: PaBlockArgs, workspace, need: int, dev) -> Optional[torch.Tensor]:
    if workspace is None:
        if need == 0:
            return None
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need or workspace.data_ptr() % 16:
        raise ValueError(f"workspace must be a contiguous, 16-byte aligned uint8 tensor of at least {need} bytes")
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    return workspace


def paged_block_attention(
    output: torch.Tensor,
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    sequence_lengths: torch.Tensor,
    block_tables: torch.Tensor,
    softmax_scale: float,
    query_sequence_length: int,
    max_sequence_length: int,
    key_scale: Optional[torch.Tensor] = None,
    value_scale: Optional[torch.Tensor] = None,
    *,
    selected_blocks: Optional[torch.Tensor] = None,
    selected_counts: Optional[torch.Tensor] = None,
    query_lens: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Decode attention over all blocks of every sequence, or over those `selected_blocks` names (logical block numbers,
    the first `selected_counts` of each list; a number outside the sequence contributes nothing, one that stands twice
    counts twice).  Writes `output` (and `lse`, the natural logarithm of every row's softmax denominator) in place and
    returns `output`; rows that see no token, and rows beyond a sequence's `query_lens` entry, become zero (lse -inf).
    Contexts are cut at `max_sequence_length` and at the block table's width.  The value rows of a sequence's tokens
    must be finite; what the cache holds behind a context does not matter."""
    plan = plan_block_attention(
        output, query, key_cache, value_cache, sequence_lengths, block_tables, softmax_scale, query_sequence_length,
        max_sequence_length, key_scale, value_scale, selected_blocks=selected_blocks, selected_counts=selected_counts,
        query_lens=query_lens, lse=lse, workspace=workspace)
    plan.run()
    return output


def key_block_bounds(
    bounds: torch.Tensor,            # [num_blocks, num_kv_heads, 2, head_size] bf16, written
    key_cache: torch.Tensor,         # [num_blocks, num_kv_heads, head_size/x, block_size, x]
    sequence_lengths: torch.Tensor,  # [num_seqs] int32
    block_tables: torch.Tensor,      # [num_seqs, max_num_blocks_per_seq] int32
    max_sequence_length: int,
    key_scale: Optional[torch.Tensor] = None,
    *,
    new_tokens: Optional[int] = None,
) -> torch.Tensor:
    """The smallest (row 0) and largest (row 1) key of every block of the sequences, over the tokens below the context
    length, rounded to bf16; NaN keys are passed over.  `new_tokens` visits only the blocks that hold each sequence's
    last so many tokens (a decode step); other blocks keep their bounds.  A block that stands in several rows has to be
    as full in each of them as far as it is visited (shared prefixes are whole blocks)."""
    a = PaBlockArgs()
    a.struct_size = C.sizeof(PaBlockArgs)
    dev = bounds.device
    _same_device(dev, key_cache=key_cache, sequence_lengths=sequence_lengths, block_tables=block_tables, key_scale=key_scale)
    _check_sequences(a, sequence_lengths, block_tables, max_sequence_length)
    _check_key_cache(a, key_cache)
    _check_scales(a, key_scale, None, False)
    _check_bounds(a, bounds)
    if tuple(bounds.shape) != (a.num_blocks, a.num_kv_heads, 2, a.head_size):
        raise ValueError(f"bounds shape {tuple(bounds.shape)} is not [{a.num_blocks}, {a.num_kv_heads}, 2, {a.head_size}]")
    if new_tokens is not None:
        if int(new_tokens) < 1:
            raise ValueError(f"new_tokens must be positive, got {new_tokens}")
        a.new_tokens = int(new_tokens)
    if not bounds.is_cuda:
        raise ValueError("key_block_bounds runs on the GPU only (there is no CPU path); got a CPU tensor")
    if a.num_seqs:
        with _on(dev):
            lib = _cabi.load_library()
            _cabi.check(lib.pa_block_bounds(C.byref(a), C.c_void_p(torch.cuda.current_stream(dev).cuda_stream)), "pa_block_bounds")
    return bounds


def select_blocks(
    query: torch.Tensor,             # [num_seqs, num_kv_heads * query_sequence_length * group, head_size] bf16
    bounds: torch.Tensor,            # [num_blocks, num_kv_heads, 2, head_size] bf16
    sequence_lengths: torch.Tensor,  # [num_seqs] int32
    block_tables: torch.Tensor,      # [num_seqs, max_num_blocks_per_seq] int32
    num_selected: int,
    block_size: int,
    query_sequence_length: int,
    max_sequence_length: int,
    *,
    first_blocks: int = 0,
    recent_blocks: Optional[int] = None,
    query_lens: Optional[torch.Tensor] = None,
    selected_blocks: Optional[torch.Tensor] = None,
    selected_counts: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The `num_selected` blocks of each (sequence, kv head) with the largest score, ascending, -1 behind the last, and
    how many there are: (int32 [num_seqs, num_kv_heads, num_selected], int32 [num_seqs, num_kv_heads]).  A block's score is
    the largest over the head's query rows of sum_d (max(q_d, 0) hi_d + min(q_d, 0) lo_d), the most that q . k can be for a
    key within the bounds; scores are ranked by their value in 64 bits, ties go to the lower block.  The first
    `first_blocks` and last `recent_blocks` blocks are always taken; `recent_blocks` defaults to, and is at least, the number of
    blocks the new tokens can lie in."""
    a = PaBlockArgs()
    a.struct_size = C.sizeof(PaBlockArgs)
    dev = query.device
    _same_device(dev, bounds=bounds, sequence_lengths=sequence_lengths, block_tables=block_tables, query_lens=query_lens,
                 selected_blocks=selected_blocks, selected_counts=selected_counts, workspace=workspace)
    _check_block_size(block_size)
    _check_sequences(a, sequence_lengths, block_tables, max_sequence_length)
    _check_bounds(a, bounds)
    a.num_blocks, a.num_kv_heads, a.block_size = bounds.shape[0], bounds.shape[1], block_size
    if a.num_blocks < 1 or a.num_kv_heads < 1:
        raise ValueError(f"bounds shape {tuple(bounds.shape)} is empty")
    _check_query(a, query, query_sequence_length, a.num_kv_heads, query_lens)
    if bounds.shape[3] != a.head_size:
        raise ValueError(f"query has head size {a.head_size}, bounds {bounds.shape[3]}")
    need_recent = 1 + (a.q_len - 1 + block_size - 1) // block_size
    recent = need_recent if recent_blocks is None else int(recent_blocks)
    if recent < need_recent:
        raise ValueError(f"recent_blocks must be at least {need_recent}: the {a.q_len} new tokens can lie in so many blocks")
    if int(num_selected) < 1 or int(first_blocks) < 0 or int(first_blocks) + recent > int(num_selected):
        raise ValueError(f"num_selected == {num_selected} does not hold first_blocks + recent_blocks == {first_blocks} + {recent}")
    if int(num_selected) * block_size > 1 << 30:
        raise ValueError(f"num_selected == {num_selected} blocks of {block_size} tokens are too many")
    a.num_selected, a.first_blocks, a.recent_blocks = int(num_selected), int(first_blocks), recent
    if not query.is_cuda:
        raise ValueError("select_blocks runs on the GPU only (there is no CPU path); got a CPU tensor")
    shape = (a.num_seqs, a.num_kv_heads)
    if selected_blocks is None:
        selected_blocks = torch.empty(shape + (a.num_selected,), dtype=torch.int32, device=dev)
    elif selected_blocks.dtype != torch.int32 or tuple(selected_blocks.shape) != shape + (a.num_selected,) or \
            (a.num_selected > 1 and selected_blocks.stride(2) != 1):
        raise ValueError(f"selected_blocks must be int32 {shape + (a.num_selected,)}, contiguous in its last dimension")
    if selected_counts is None:
        selected_counts = torch.empty(shape, dtype=torch.int32, device=dev)
    elif selected_counts.dtype != torch.int32 or tuple(selected_counts.shape) != shape or \
            (shape[1] > 1 and selected_counts.stride(1) != 1):
        raise ValueError(f"selected_counts must be int32 {shape}, dense over the heads")
    if a.num_seqs:
        a.selected_blocks, a.selected_counts = selected_blocks.data_ptr(), selected_counts.data_ptr()
        a.stride_sel_s, a.stride_sel_h = selected_blocks.stride(0), selected_blocks.stride(1)
        a.stride_cnt_s = selected_counts.stride(0)
        keep = _give_workspace(a, workspace, _workspace_bytes("pa_select_blocks_workspace_bytes", a), dev)
        with _on(dev):
            lib = _cabi.load_library()
            _cabi.check(lib.pa_select_blocks(C.byref(a), C.c_void_p(torch.cuda.current_stream(dev).cuda_stream)), "pa_select_blocks")
        del keep
    return selected_blocks, selected_counts
