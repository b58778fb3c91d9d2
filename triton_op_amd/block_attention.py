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

import ctypes as C
import functools
import struct
from typing import Optional, Tuple

import torch

from . import _cabi
from ._cabi import PaBlockArgs
from .kv_cache import FP8_DTYPE, _check_written, _current_raw_stream, _strides

_SUPPORTED_BLOCK_SIZES = (16, 64, 1024)
_SUPPORTED_HEAD_SIZES = (64, 128, 256)

# PaBlockArgs in one go, in the order of its fields (filling some 50 attributes of a ctypes structure takes longer than
# the kernels of a small call)
_PACK = struct.Struct("<Ii14Q16ifi20q")
_SIZE = C.sizeof(PaBlockArgs)
assert _PACK.size == _SIZE


def _check_devices(index: int, dev: torch.device, tensors: dict) -> None:
    for name, t in tensors.items():
        if t is not None and (t.get_device() != index or (index < 0 and t.device != dev)):
            raise ValueError(f"{name} is on {t.device}, the call on {dev}")


def _launch(name: str, args: PaBlockArgs, index: int, stream: Optional[int] = None) -> None:
    """Calls an entry point of the library on torch's current stream of device `index`, with that device current."""
    if index == torch.cuda.current_device():
        if stream is None:
            stream = _current_raw_stream(index)
        rc = getattr(_cabi.load_library(), name)(C.byref(args), stream)
        if rc:
            _cabi.check(rc, name)
    else:
        with torch.cuda.device(index):
            _launch(name, args, index, stream)


def _check_sequences(lens, tables) -> Tuple[int, int, int]:
    """(number of sequences, entries of a table row, stride of the rows)"""
    if lens.dtype is not torch.int32 or tables.dtype is not torch.int32:
        raise ValueError("sequence_lengths and block_tables must be int32")
    shape = tables.shape
    if len(shape) != 2 or lens.numel() != shape[0] or shape[1] < 1:
        raise ValueError("sequence_lengths / block_tables do not have one row per sequence")
    row, col = tables.stride()
    if not lens.is_contiguous() or (col != 1 and shape[1] > 1):
        raise ValueError("sequence_lengths and the rows of block_tables must be contiguous")
    return shape[0], shape[1], row


def _check_query(query, q_len: int, num_kv_heads: int, num_seqs: int, query_lens) -> Tuple[int, int, int, int]:
    """(query rows per kv head and new token, head size, strides)"""
    if query.dim() != 3:
        raise ValueError(f"Expected 3D query tensor, but got shape {tuple(query.shape)}")
    if query.dtype is not torch.bfloat16:
        raise ValueError(f"query tensor only supports dtype bfloat16, but got {query.dtype}")
    seqs, rows, head_size = query.shape
    if q_len < 1 or rows == 0 or rows % (q_len * num_kv_heads):
        raise ValueError(f"query.shape[1]={rows} is not num_kv_heads*query_sequence_length*group ({num_kv_heads}*{q_len}*G)")
    if rows // num_kv_heads > 64:
        raise ValueError(f"{rows // num_kv_heads} query rows per kv head exceed the maximum of 64")
    if seqs != num_seqs:
        raise ValueError("sequence_lengths / block_tables do not have one row per sequence")
    if head_size not in _SUPPORTED_HEAD_SIZES:
        raise ValueError(f"head_size == {head_size} is not supported (64, 128 or 256)")
    st = query.stride()
    if st[0] % 8 or st[1] % 8:
        st = _strides(query)
    if st[2] != 1 or st[0] % 8 or st[1] % 8 or query.data_ptr() % 16:
        raise ValueError("query rows must be dense and 16-byte aligned")
    if query_lens is not None and (query_lens.dtype is not torch.int32 or query_lens.numel() != seqs or not query_lens.is_contiguous()):
        raise ValueError("query_lens must be contiguous int32 [num_seqs]")
    return rows // (q_len * num_kv_heads), head_size, st[0], st[1]


def _check_block_size(block_size: int) -> None:
    if block_size not in _SUPPORTED_BLOCK_SIZES:
        raise ValueError(f"kv_block_size == {block_size} not in {list(_SUPPORTED_BLOCK_SIZES)}")


def _check_key_cache(key_cache):
    """(dtype code, elements per 16 bytes, blocks, kv heads, block size, head size, strides of the first three dimensions)"""
    shape = key_cache.shape
    if len(shape) != 5:
        raise ValueError(f"Expected 5D key_cache tensor, but got shape {tuple(shape)}")
    if key_cache.dtype is FP8_DTYPE:
        code, x = _cabi.PA_DTYPE_FP8_E4M3FN, 16
    elif key_cache.dtype is torch.bfloat16:
        code, x = _cabi.PA_DTYPE_BF16, 8
    else:
        raise ValueError(f"key_cache tensor only supports dtype bfloat16 or float8_e4m3fn, but got {key_cache.dtype}")
    blocks, heads, chunks, bs, inner = shape
    _check_block_size(bs)
    if inner != x or chunks * x not in _SUPPORTED_HEAD_SIZES or blocks < 1 or heads < 1:
        raise ValueError(f"key_cache shape {tuple(shape)} is not [blocks, kv_heads, head_size//{x}, bs, {x}] "
                         "with a head size of 64, 128 or 256")
    s0, s1, s2, s3, s4 = key_cache.stride()
    if s0 % x or s1 % x:
        s0, s1 = _strides(key_cache)[:2]
    if s4 != 1 or s3 != x or s0 % x or s1 % x or s2 % x or key_cache.data_ptr() % 16:
        raise ValueError("the innermost dimensions of key_cache must be dense and 16-byte aligned")
    return code, x, blocks, heads, bs, chunks * x, s0, s1, s2


def _check_scales(code: int, blocks: int, heads: int, bs: int, key_scale, value_scale, both: bool) -> Tuple[int, int, int]:
    """(quantisation mode, strides over blocks and heads)"""
    if both and (key_scale is None) != (value_scale is None):
        raise ValueError("key_scale and value_scale must be given together")
    if key_scale is None:
        return _cabi.PA_QUANT_NONE, 0, 0
    if code != _cabi.PA_DTYPE_FP8_E4M3FN:
        raise ValueError("scales need an FP8 cache")
    if key_scale.dtype is not torch.float32 or (both and value_scale.dtype is not torch.float32):
        raise ValueError("key_scale / value_scale tensors only support dtype == torch.float32")
    shape = tuple(key_scale.shape)
    if both and (shape != tuple(value_scale.shape) or (key_scale.stride() != value_scale.stride() and _strides(key_scale) != _strides(value_scale))):
        raise ValueError("key and value scales must have the same shape and strides")
    if shape == ():
        return _cabi.PA_QUANT_PER_TENSOR, 0, 0
    st = key_scale.stride()
    if shape == (blocks, heads, 1, 1):
        return _cabi.PA_QUANT_PER_BLOCK, st[0], st[1]
    if shape != (blocks, heads, bs, 1):
        raise ValueError(f"Expected scales of shape [], [{blocks}, {heads}, 1, 1] or [{blocks}, {heads}, {bs}, 1], got {shape}")
    if st[0] % 4 or st[1] % 4:
        st = _strides(key_scale)
    if st[2] != 1 or st[0] % 4 or st[1] % 4 or key_scale.data_ptr() % 16 or (both and value_scale.data_ptr() % 16):
        raise ValueError("per-token scales must be dense over tokens and 16-byte aligned")
    return _cabi.PA_QUANT_PER_TOKEN, st[0], st[1]


def _check_bounds(bounds) -> Tuple[int, int]:
    """strides over blocks and heads"""
    shape = bounds.shape
    if bounds.dtype is not torch.bfloat16 or len(shape) != 4 or shape[2] != 2:
        raise ValueError("bounds must be bfloat16 [num_blocks, num_kv_heads, 2, head_size]")
    s0, s1, s2, s3 = bounds.stride()
    if s0 % 8 or s1 % 8:
        s0, s1 = _strides(bounds)[:2]
    if s3 != 1 or s2 != shape[3] or s0 % 8 or s1 % 8 or bounds.data_ptr() % 16:
        raise ValueError("the two bounds of a (block, head) must be dense and 16-byte aligned")
    return s0, s1


@functools.lru_cache(maxsize=4096)
def _attention_workspace(num_seqs, heads, group, q_len, head_size, bs, code, width, longest, num_selected) -> int:
    """pa_block_attention_workspace_bytes, a pure function of these sizes."""
    aligned = 1 << 12  # (an address that passes the library's checks and is not followed)
    a = PaBlockArgs(struct_size=_SIZE, output=aligned, query=aligned, key_cache=aligned, value_cache=aligned, context_lens=aligned,
                    block_tables=aligned, num_seqs=num_seqs, num_kv_heads=heads, group_size=group, q_len=q_len, head_size=head_size,
                    block_size=bs, kv_dtype=code, num_blocks=1, table_width=width, max_context_len=longest,
                    kv_quant_mode=_cabi.PA_QUANT_NONE, selected_blocks=aligned if num_selected else None, num_selected=num_selected)
    return _workspace_bytes("pa_block_attention_workspace_bytes", a)


@functools.lru_cache(maxsize=4096)
def _select_workspace(num_seqs, heads, group, q_len, head_size, bs, width, longest) -> int:
    """pa_select_blocks_workspace_bytes, a pure function of these sizes."""
    aligned = 1 << 12
    a = PaBlockArgs(struct_size=_SIZE, query=aligned, context_lens=aligned, block_tables=aligned, bounds=aligned, selected_blocks=aligned,
                    selected_counts=aligned, num_seqs=num_seqs, num_kv_heads=heads, group_size=group, q_len=q_len, head_size=head_size,
                    block_size=bs, num_blocks=1, table_width=width, max_context_len=longest, num_selected=1)
    return _workspace_bytes("pa_select_blocks_workspace_bytes", a)


def _workspace_bytes(name: str, a: PaBlockArgs) -> int:
    need = getattr(_cabi.load_library(), name)(C.byref(a))
    if need < 0:
        _cabi.check(int(need), name)
    return need


def _give_workspace(workspace, need: int, dev) -> Optional[torch.Tensor]:
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    if workspace.dtype is not torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need or workspace.data_ptr() % 16:
        raise ValueError(f"workspace must be a contiguous, 16-byte aligned uint8 tensor of at least {need} bytes")
    return workspace


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


class BlockAttentionPlan:
    """A validated call: the filled C struct plus the tensors it points to (kept alive).  `run()` enqueues it on a
    stream; it allocates nothing and can be replayed, and captured.  Plans that may overlap on the GPU need a
    workspace each (a plan made without one has its own).  Keep the plan until its work has run: a workspace of its own
    goes back to the allocator with it."""

    def __init__(self, args: PaBlockArgs, keep, output):
        self.args, self._keep, self.output = args, keep, output
        self._index = output.get_device()

    def run(self, stream: Optional[int] = None) -> None:
        if self.args.num_seqs:
            _launch("pa_block_attention", self.args, self._index, stream)


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
    dev, index = output.device, output.get_device()
    _check_devices(index, dev, dict(
        query=query, key_cache=key_cache, value_cache=value_cache, sequence_lengths=sequence_lengths, block_tables=block_tables,
        key_scale=key_scale, value_scale=value_scale, selected_blocks=selected_blocks, selected_counts=selected_counts,
        query_lens=query_lens, lse=lse, workspace=workspace))
    num_seqs, width, st_bt = _check_sequences(sequence_lengths, block_tables)
    code, x, blocks, heads, bs, head_size, st_kb, st_kh, st_kc = _check_key_cache(key_cache)
    q_len, longest = int(query_sequence_length), max(0, min(int(max_sequence_length), width * bs))
    group, q_head_size, st_qs, st_qh = _check_query(query, q_len, heads, num_seqs, query_lens)
    if q_head_size != head_size:
        raise ValueError(f"query has head size {q_head_size}, key_cache {head_size}")
    if output.shape != query.shape or output.dtype is not torch.bfloat16:
        raise ValueError(f"output must be bfloat16 {tuple(query.shape)}, got {output.dtype} {tuple(output.shape)}")
    st_os, st_oh, st_od = output.stride()
    if st_os % 4 or st_oh % 4:
        st_os, st_oh, _ = _strides(output)
    if st_od != 1 or st_os % 4 or st_oh % 4 or output.data_ptr() % 8:
        raise ValueError("output rows must be dense and 8-byte aligned")
    # ---- value cache ---------------------------------------------------------------------------------------------------
    if value_cache.dtype is not key_cache.dtype:
        raise ValueError(f"value_cache dtype {value_cache.dtype} differs from key_cache dtype {key_cache.dtype}")
    v_transposed = value_cache.dim() == 5
    if value_cache.shape != ((blocks, heads, bs // x, head_size, x) if v_transposed else (blocks, heads, head_size, bs)):
        raise ValueError(f"value_cache shape {tuple(value_cache.shape)} is not [blocks, kv_heads, D, bs] or, transposed, "
                         f"[blocks, kv_heads, bs/{x}, D, {x}] of the key cache")
    st_v = value_cache.stride()
    if st_v[0] % x or st_v[1] % x or st_v[2] % x:
        st_v = _strides(value_cache)
    if st_v[-1] != 1 or (v_transposed and st_v[3] != x) or st_v[0] % x or st_v[1] % x or st_v[2] % x or value_cache.data_ptr() % 16:
        raise ValueError("the innermost dimensions of value_cache must be dense and 16-byte aligned")
    mode, st_sb, st_sh = _check_scales(code, blocks, heads, bs, key_scale, value_scale, True)
    # ---- the list ----------------------------------------------------------------------------------------------------------
    num_selected = st_ls = st_lh = st_cs = st_lse = 0
    if selected_blocks is not None:
        shape = selected_blocks.shape
        if selected_blocks.dtype is not torch.int32 or len(shape) != 3 or shape[0] != num_seqs or shape[1] != heads or shape[2] < 1:
            raise ValueError(f"selected_blocks must be int32 [{num_seqs}, {heads}, k]")
        num_selected = shape[2]
        st_ls, st_lh, st_lk = selected_blocks.stride()
        if num_selected > 1 and st_lk != 1:
            raise ValueError("selected_blocks must be contiguous in its last dimension")
    if selected_counts is not None:
        if selected_blocks is None:
            raise ValueError("selected_counts needs selected_blocks")
        if selected_counts.dtype is not torch.int32 or selected_counts.shape != (num_seqs, heads) or (heads > 1 and selected_counts.stride(1) != 1):
            raise ValueError(f"selected_counts must be int32 [{num_seqs}, {heads}], dense over the heads")
        st_cs = selected_counts.stride(0)
    if lse is not None:
        if lse.dtype is not torch.float32 or lse.shape != query.shape[:2] or (lse.stride(1) != 1 and lse.shape[1] > 1):
            raise ValueError(f"lse must be float32 {tuple(query.shape[:2])}, dense over the rows")
        st_lse = lse.stride(0)
    if not (st_os and st_oh and (st_lse or lse is None)):
        _check_written(output=output, lse=lse)
    if not output.is_cuda:
        raise ValueError("paged_block_attention runs on the GPU only (there is no CPU path); got a CPU tensor")
    if num_seqs:
        need = _attention_workspace(num_seqs, heads, group, q_len, head_size, bs, code, width, longest, num_selected)
        workspace = _give_workspace(workspace, need, dev)
    args = PaBlockArgs.from_buffer_copy(_PACK.pack(
        _SIZE, 0,
        output.data_ptr(), query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), _ptr(key_scale), _ptr(value_scale),
        sequence_lengths.data_ptr(), block_tables.data_ptr(), _ptr(query_lens), 0, _ptr(selected_blocks), _ptr(selected_counts), _ptr(lse),
        _ptr(workspace),
        num_seqs, heads, group, q_len, head_size, bs, blocks, width, longest, code, mode, v_transposed, num_selected, 0, 0, 0,
        softmax_scale, 0,
        st_os, st_oh, st_qs, st_qh, st_kb, st_kh, st_kc, st_v[0], st_v[1], st_v[2], st_sb, st_sh, st_bt, 0, 0,
        st_ls, st_lh, st_cs, st_lse, 0 if workspace is None else workspace.numel()))
    keep = (output, query, key_cache, value_cache, sequence_lengths, block_tables, key_scale, value_scale,
            selected_blocks, selected_counts, query_lens, lse, workspace)
    return BlockAttentionPlan(args, keep, output)


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
    must be finite, and so must the scales, of either sign; what the cache holds behind a context does not matter."""
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
    dev, index = bounds.device, bounds.get_device()
    _check_devices(index, dev, dict(key_cache=key_cache, sequence_lengths=sequence_lengths, block_tables=block_tables, key_scale=key_scale))
    num_seqs, width, st_bt = _check_sequences(sequence_lengths, block_tables)
    code, _, blocks, heads, bs, head_size, st_kb, st_kh, st_kc = _check_key_cache(key_cache)
    mode, st_sb, st_sh = _check_scales(code, blocks, heads, bs, key_scale, None, False)
    st_bb, st_bh = _check_bounds(bounds)
    if bounds.shape != (blocks, heads, 2, head_size):
        raise ValueError(f"bounds shape {tuple(bounds.shape)} is not [{blocks}, {heads}, 2, {head_size}]")
    if not (st_bb and st_bh):
        _check_written(bounds=bounds)
    new, longest = 0 if new_tokens is None else int(new_tokens), max(0, min(int(max_sequence_length), width * bs))
    if new_tokens is not None and new < 1:
        raise ValueError(f"new_tokens must be positive, got {new_tokens}")
    if not bounds.is_cuda:
        raise ValueError("key_block_bounds runs on the GPU only (there is no CPU path); got a CPU tensor")
    if num_seqs:
        args = PaBlockArgs.from_buffer_copy(_PACK.pack(
            _SIZE, 0,
            0, 0, key_cache.data_ptr(), 0, _ptr(key_scale), 0, sequence_lengths.data_ptr(), block_tables.data_ptr(), 0, bounds.data_ptr(), 0, 0, 0, 0,
            num_seqs, heads, 0, 0, head_size, bs, blocks, width, longest, code, mode, 0, 0, 0, 0, min(new, 1 << 30),
            0.0, 0,
            0, 0, 0, 0, st_kb, st_kh, st_kc, 0, 0, 0, st_sb, st_sh, st_bt, st_bb, st_bh, 0, 0, 0, 0, 0))
        _launch("pa_block_bounds", args, index)
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
    blocks the new tokens can lie in.  A list is decided in 32 bits with a bound of their error, and many times slower where
    that does not decide it: more than 65536 blocks, a bound that is no finite number, a table entry outside the cache, a
    sequence without a query row, or one block of far larger keys than the others' (take the first with `first_blocks`)."""
    dev, index = query.device, query.get_device()
    _check_devices(index, dev, dict(
        bounds=bounds, sequence_lengths=sequence_lengths, block_tables=block_tables, query_lens=query_lens, selected_blocks=selected_blocks,
        selected_counts=selected_counts, workspace=workspace))
    _check_block_size(block_size)
    num_seqs, width, st_bt = _check_sequences(sequence_lengths, block_tables)
    st_bb, st_bh = _check_bounds(bounds)
    blocks, heads, _, head_size = bounds.shape
    if blocks < 1 or heads < 1:
        raise ValueError(f"bounds shape {tuple(bounds.shape)} is empty")
    q_len, longest = int(query_sequence_length), max(0, min(int(max_sequence_length), width * block_size))
    k, first = int(num_selected), int(first_blocks)
    group, q_head_size, st_qs, st_qh = _check_query(query, q_len, heads, num_seqs, query_lens)
    if q_head_size != head_size:
        raise ValueError(f"query has head size {q_head_size}, bounds {head_size}")
    need_recent = 1 + (q_len - 1 + block_size - 1) // block_size
    recent = need_recent if recent_blocks is None else int(recent_blocks)
    if recent < need_recent:
        raise ValueError(f"recent_blocks must be at least {need_recent}: the {q_len} new tokens can lie in so many blocks")
    if k < 1 or first < 0 or first + recent > k:
        raise ValueError(f"num_selected == {num_selected} does not hold first_blocks + recent_blocks == {first_blocks} + {recent}")
    if k * block_size > 1 << 30:
        raise ValueError(f"num_selected == {num_selected} blocks of {block_size} tokens are too many")
    if selected_blocks is not None or selected_counts is not None:
        _check_written(selected_blocks=selected_blocks, selected_counts=selected_counts)
    if not query.is_cuda:
        raise ValueError("select_blocks runs on the GPU only (there is no CPU path); got a CPU tensor")
    if selected_blocks is None:
        selected_blocks = torch.empty((num_seqs, heads, k), dtype=torch.int32, device=dev)
    elif selected_blocks.dtype is not torch.int32 or selected_blocks.shape != (num_seqs, heads, k) or (k > 1 and selected_blocks.stride(2) != 1):
        raise ValueError(f"selected_blocks must be int32 {(num_seqs, heads, k)}, contiguous in its last dimension")
    if selected_counts is None:
        selected_counts = torch.empty((num_seqs, heads), dtype=torch.int32, device=dev)
    elif selected_counts.dtype is not torch.int32 or selected_counts.shape != (num_seqs, heads) or (heads > 1 and selected_counts.stride(1) != 1):
        raise ValueError(f"selected_counts must be int32 {(num_seqs, heads)}, dense over the heads")
    if num_seqs:
        workspace = _give_workspace(workspace, _select_workspace(num_seqs, heads, group, q_len, head_size, block_size, width, longest), dev)
        st_ls, st_lh, _ = selected_blocks.stride()
        args = PaBlockArgs.from_buffer_copy(_PACK.pack(
            _SIZE, 0,
            0, query.data_ptr(), 0, 0, 0, 0, sequence_lengths.data_ptr(), block_tables.data_ptr(), _ptr(query_lens), bounds.data_ptr(),
            selected_blocks.data_ptr(), selected_counts.data_ptr(), 0, workspace.data_ptr(),
            num_seqs, heads, group, q_len, head_size, block_size, blocks, width, longest, 0, _cabi.PA_QUANT_NONE, 0, k, first, recent, 0,
            0.0, 0,
            0, 0, st_qs, st_qh, 0, 0, 0, 0, 0, 0, 0, 0, st_bt, st_bb, st_bh, st_ls, st_lh, selected_counts.stride(0), 0, workspace.numel()))
        _launch("pa_select_blocks", args, index)
    return selected_blocks, selected_counts
