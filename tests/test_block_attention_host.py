"""CPU-side tests of the block-granular operators: what the entry points and the C ABI refuse, the layout of the struct, the
cut of the token axis and the workspace sizes, and the oracle against torch."""
import ctypes as C
import math
import os
import re

import pytest
import torch

import triton_op_amd as T
from oracle import block_oracle as O
from triton_op_amd import _cabi

FP8 = torch.float8_e4m3fn
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def _attention(**over):
    kw = dict(output=_z(2, 8, 128, dtype=torch.bfloat16), query=_z(2, 8, 128, dtype=torch.bfloat16), key_cache=_z(9, 2, 8, 16, 16).to(FP8),
              value_cache=_z(9, 2, 128, 16).to(FP8), sequence_lengths=torch.tensor([40, 20], dtype=torch.int32),
              block_tables=_z(2, 3, dtype=torch.int32), softmax_scale=0.1, query_sequence_length=1, max_sequence_length=40,
              key_scale=_z(9, 2, 1, 1), value_scale=_z(9, 2, 1, 1))
    kw.update(over)
    return kw


@pytest.mark.parametrize("over,msg", [
    (dict(), "GPU only"),
    (dict(key_scale=None, value_scale=None), "GPU only"),
    (dict(key_scale=_z(9, 2, 16, 1), value_scale=_z(9, 2, 16, 1)), "GPU only"),
    (dict(selected_blocks=_z(2, 2, 5, dtype=torch.int32), selected_counts=_z(2, 2, dtype=torch.int32), lse=_z(2, 8)), "GPU only"),
    (dict(query=_z(2, 8, 128)), "bfloat16"),
    (dict(query=_z(2, 128, dtype=torch.bfloat16)), "3D query"),
    (dict(output=_z(2, 8, 128)), "output must be bfloat16"),
    (dict(output=_z(2, 4, 128, dtype=torch.bfloat16)), "output must be bfloat16"),
    (dict(query_sequence_length=3), "is not num_kv_heads"),
    (dict(query=_z(2, 130, 128, dtype=torch.bfloat16), output=_z(2, 130, 128, dtype=torch.bfloat16)), "maximum of 64"),
    (dict(query=_z(2, 8, 64, dtype=torch.bfloat16), output=_z(2, 8, 64, dtype=torch.bfloat16)), "head size"),
    (dict(query=_z(2, 8, 130, dtype=torch.bfloat16)[..., :128]), "16-byte aligned"),
    (dict(key_cache=_z(9, 2, 8, 16)), "5D key_cache"),
    (dict(key_cache=_z(9, 2, 8, 16, 16)), "bfloat16 or float8"),
    (dict(key_cache=_z(9, 2, 8, 32, 16).to(FP8)), "kv_block_size"),
    (dict(key_cache=_z(9, 2, 6, 16, 16).to(FP8)), "head size"),
    (dict(value_cache=_z(9, 2, 128, 16, dtype=torch.bfloat16)), "differs from key_cache"),
    (dict(value_cache=_z(8, 2, 128, 16).to(FP8)), "value_cache shape"),
    (dict(value_cache=_z(9, 2, 2, 128, 16).to(FP8)), "value_cache shape"),
    (dict(value_scale=None), "given together"),
    (dict(key_scale=_z(9, 2, 1, 1, dtype=torch.float64)), "float32"),
    (dict(key_scale=_z(9, 2, 1)), "same shape"),
    (dict(key_scale=_z(9, 1, 1, 1), value_scale=_z(9, 1, 1, 1)), "Expected scales"),
    (dict(key_cache=_z(9, 2, 16, 16, 8, dtype=torch.bfloat16), value_cache=_z(9, 2, 128, 16, dtype=torch.bfloat16)), "FP8 cache"),
    (dict(sequence_lengths=torch.tensor([40, 20])), "int32"),
    (dict(block_tables=_z(3, 3, dtype=torch.int32)), "one row per sequence"),
    (dict(sequence_lengths=torch.zeros(3, dtype=torch.int32), block_tables=_z(3, 3, dtype=torch.int32)), "one row per sequence"),
    (dict(block_tables=_z(2, 6, dtype=torch.int32)[:, ::2]), "contiguous"),
    (dict(query_lens=torch.zeros(2)), "query_lens"),
    (dict(query_lens=torch.zeros(3, dtype=torch.int32)), "query_lens"),
    (dict(selected_blocks=_z(2, 2, 0, dtype=torch.int32)), "selected_blocks must be"),
    (dict(selected_blocks=_z(2, 3, 4, dtype=torch.int32)), "selected_blocks must be"),
    (dict(selected_blocks=torch.zeros(2, 2, 4, dtype=torch.int64)), "selected_blocks must be"),
    (dict(selected_blocks=_z(2, 2, 8, dtype=torch.int32)[..., ::2]), "contiguous in its last"),
    (dict(selected_counts=_z(2, 2, dtype=torch.int32)), "needs selected_blocks"),
    (dict(selected_blocks=_z(2, 2, 4, dtype=torch.int32), selected_counts=_z(2, 3, dtype=torch.int32)), "selected_counts must be"),
    (dict(lse=_z(2, 9)), "lse must be"),
    (dict(lse=_z(2, 8, dtype=torch.float64)), "lse must be"),
    (dict(lse=torch.zeros(2, 8, device="meta")), "lse is on meta"),
])
def test_attention_refuses(over, msg):
    with pytest.raises(ValueError, match=msg):
        T.paged_block_attention(**_attention(**over))


def _bounds(**over):
    kw = dict(bounds=_z(9, 2, 2, 128, dtype=torch.bfloat16), key_cache=_z(9, 2, 8, 16, 16).to(FP8),
              sequence_lengths=torch.tensor([40, 20], dtype=torch.int32), block_tables=_z(2, 3, dtype=torch.int32), max_sequence_length=40,
              key_scale=_z(9, 2, 1, 1))
    kw.update(over)
    return kw


@pytest.mark.parametrize("over,msg", [
    (dict(), "GPU only"),
    (dict(key_scale=torch.tensor(1.0), new_tokens=3), "GPU only"),
    (dict(bounds=_z(9, 2, 2, 128)), "bounds must be"),
    (dict(bounds=_z(9, 2, 1, 128, dtype=torch.bfloat16)), "bounds must be"),
    (dict(bounds=_z(8, 2, 2, 128, dtype=torch.bfloat16)), "bounds shape"),
    (dict(bounds=_z(9, 2, 2, 64, dtype=torch.bfloat16)), "bounds shape"),
    (dict(bounds=_z(9, 2, 2, 256, dtype=torch.bfloat16)[..., ::2]), "dense"),
    (dict(new_tokens=0), "new_tokens must be positive"),
    (dict(key_scale=_z(9, 2, 2, 1)), "Expected scales"),
    (dict(block_tables=torch.zeros(2, 3, dtype=torch.int32, device="meta")), "block_tables is on meta"),
])
def test_bounds_refuses(over, msg):
    with pytest.raises(ValueError, match=msg):
        T.key_block_bounds(**_bounds(**over))


def _select(**over):
    kw = dict(query=_z(2, 8, 128, dtype=torch.bfloat16), bounds=_z(9, 2, 2, 128, dtype=torch.bfloat16),
              sequence_lengths=torch.tensor([40, 20], dtype=torch.int32), block_tables=_z(2, 3, dtype=torch.int32), num_selected=2, block_size=16,
              query_sequence_length=1, max_sequence_length=40)
    kw.update(over)
    return kw


@pytest.mark.parametrize("over,msg", [
    (dict(), "GPU only"),
    (dict(num_selected=0), "does not hold"),
    (dict(first_blocks=2), "does not hold"),
    (dict(first_blocks=-1), "does not hold"),
    (dict(recent_blocks=0), "recent_blocks must be at least 1"),
    (dict(query_sequence_length=2, recent_blocks=1), "recent_blocks must be at least 2"),
    (dict(query_sequence_length=2, num_selected=1), "does not hold"),
    (dict(block_size=32), "kv_block_size"),
    (dict(num_selected=1 << 28), "too many"),
    (dict(bounds=_z(9, 2, 2, 64, dtype=torch.bfloat16)), "head size"),
    (dict(bounds=_z(9, 3, 2, 128, dtype=torch.bfloat16)), "is not num_kv_heads"),
    (dict(query_lens=_z(1, dtype=torch.int32)), "query_lens"),
    (dict(query=_z(2, 8, 96, dtype=torch.bfloat16)), "not supported"),
])
def test_select_refuses(over, msg):
    with pytest.raises(ValueError, match=msg):
        T.select_blocks(**_select(**over))


def test_write_refuses_what_its_scales_do_not_fit(monkeypatch):
    from triton_op_amd import kv_cache as KC

    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    key = _z(3, 2, 128, dtype=torch.bfloat16)
    good = dict(key=key, value=key, key_cache=_z(9, 2, 8, 16, 16).to(FP8), value_cache=_z(9, 2, 128, 16).to(FP8),
                slot_mapping=torch.zeros(3, dtype=torch.int64), key_scale=_z(9, 2, 1, 1), value_scale=_z(9, 2, 1, 1))
    for over, msg in ((dict(value_scale=_z(9, 2, 16, 1)), "same shape"), (dict(key_scale=_z(8, 2, 1, 1), value_scale=_z(8, 2, 1, 1)), "per-token scales"),
                      (dict(value_scale=_z(2, 9, 1, 1).transpose(0, 1)), "same strides"),
                      (dict(value_cache=_z(8, 2, 128, 16).to(FP8)), "value_cache 8"),
                      (dict(key_cache=_z(9, 2, 16, 16, 8, dtype=torch.bfloat16), value_cache=_z(9, 2, 128, 16, dtype=torch.bfloat16)), "FP8 cache")):
        with pytest.raises(ValueError, match=msg):
            KC.kv_cache_write(**{**good, **over})


@pytest.mark.parametrize("call,over", [
    (_attention, dict(output=_z(1, 8, 128, dtype=torch.bfloat16).expand(2, 8, 128))),
    (_attention, dict(output=_z(2, 1, 128, dtype=torch.bfloat16).expand(2, 8, 128))),
    (_attention, dict(lse=_z(1, 8).expand(2, 8))),
    (_bounds, dict(bounds=_z(9, 1, 2, 128, dtype=torch.bfloat16).expand(9, 2, 2, 128))),
    (_bounds, dict(bounds=_z(1, 2, 2, 128, dtype=torch.bfloat16).expand(9, 2, 2, 128))),
    (_select, dict(selected_blocks=_z(2, 1, 2, dtype=torch.int32).expand(2, 2, 2))),
    (_select, dict(selected_counts=_z(1, 2, dtype=torch.int32).expand(2, 2))),
])
def test_written_tensors_must_not_be_expanded(call, over):
    """Several results for one place: what is left there would depend on which workgroup comes last."""
    entry = {_attention: T.paged_block_attention, _bounds: T.key_block_bounds, _select: T.select_blocks}[call]
    with pytest.raises(ValueError, match="must not be an expanded tensor"):
        entry(**call(**over))


def test_expanded_tensors_that_are_only_read_are_fine():
    one = _z(1, 1, 1, 1)
    for call, entry, over in (
            (_attention, T.paged_block_attention, dict(key_scale=one.expand(9, 2, 1, 1), value_scale=one.expand(9, 2, 1, 1))),
            (_attention, T.paged_block_attention, dict(block_tables=_z(1, 3, dtype=torch.int32).expand(2, 3), lse=_z(2, 8),
                                                       selected_blocks=_z(2, 1, 5, dtype=torch.int32).expand(2, 2, 5))),
            (_bounds, T.key_block_bounds, dict(key_scale=one.expand(9, 2, 1, 1))),
            (_select, T.select_blocks, dict(bounds=_z(1, 2, 2, 128, dtype=torch.bfloat16).expand(9, 2, 2, 128)))):
        with pytest.raises(ValueError, match="GPU only"):
            entry(**call(**over))


def _odd(t, *dims):
    """The tensor with strides that mean nothing (odd ones) in dimensions of size 1."""
    st = list(t.stride())
    for i in dims:
        assert t.shape[i] == 1
        st[i] = 7
    return t.as_strided(t.shape, st)


def test_strides_of_dimensions_of_size_one_mean_nothing():
    b16 = dict(dtype=torch.bfloat16)
    one = dict(output=_odd(_z(1, 1, 128, **b16), 0, 1), query=_odd(_z(1, 1, 128, **b16), 0, 1), key_cache=_odd(_z(1, 1, 8, 16, 16).to(FP8), 0, 1),
               value_cache=_odd(_z(1, 1, 1, 128, 16).to(FP8), 0, 1, 2), sequence_lengths=torch.tensor([9], dtype=torch.int32),
               block_tables=_odd(_z(1, 1, dtype=torch.int32), 0, 1), key_scale=_odd(_z(1, 1, 16, 1), 0, 1), value_scale=_odd(_z(1, 1, 16, 1), 0, 1),
               lse=_odd(_z(1, 1), 0, 1), selected_blocks=_odd(_z(1, 1, 1, dtype=torch.int32), 0, 1, 2),
               selected_counts=_odd(_z(1, 1, dtype=torch.int32), 0, 1))
    for over in ({}, dict(key_scale=_odd(_z(1, 1, 1, 1), 0, 1), value_scale=_odd(_z(1, 1, 1, 1), 0, 1, 2))):
        with pytest.raises(ValueError, match="GPU only"):
            T.paged_block_attention(**_attention(**{**one, **over}))
    box = _odd(_z(1, 1, 2, 128, **b16), 0, 1)
    with pytest.raises(ValueError, match="GPU only"):
        T.key_block_bounds(**_bounds(bounds=box, **{n: one[n] for n in ("key_cache", "sequence_lengths", "block_tables", "key_scale")}))
    with pytest.raises(ValueError, match="GPU only"):
        T.select_blocks(**_select(bounds=box, num_selected=1, **{n: one[n] for n in ("query", "sequence_lengths", "block_tables")}))


def test_write_refuses_scales_that_share_their_memory(monkeypatch):
    """A head's scale decides its codes: heads (or K and V) that write one scale each into the same place leave codes without theirs."""
    from triton_op_amd import kv_cache as KC

    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    key = _z(3, 2, 128, dtype=torch.bfloat16)
    good = dict(key=key, value=key, key_cache=_z(9, 2, 8, 16, 16).to(FP8), value_cache=_z(9, 2, 128, 16).to(FP8),
                slot_mapping=torch.zeros(3, dtype=torch.int64), key_scale=_z(9, 2, 1, 1), value_scale=_z(9, 2, 1, 1))
    per_block = dict(key_scale=_z(9, 1, 1, 1).expand(9, 2, 1, 1), value_scale=_z(9, 1, 1, 1).expand(9, 2, 1, 1))
    same = dict(key_scale=good["key_scale"], value_scale=good["key_scale"])
    cache = dict(key_cache=_z(1, 2, 8, 16, 16).to(FP8).expand(9, 2, 8, 16, 16))
    for over, msg in ((per_block, "expanded"), (same, "same memory"), (cache, "expanded")):
        with pytest.raises(ValueError, match=msg):
            KC.kv_cache_write(**{**good, **over})


def test_struct_matches_the_header(pa_lib):
    with open(os.path.join(ROOT, "include", "pa_decode.h")) as f:
        body = re.search(r"typedef struct PaBlockArgs \{(.*?)\} PaBlockArgs;", f.read(), re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for decl in body.split(";"):
        decl = decl.strip()
        if decl:
            names += [n.strip().lstrip("*") for n in re.sub(r"^(const\s+)?[a-z0-9_]+\s*\**", "", decl, count=1).split(",")]
    assert names == [f[0] for f in _cabi.PaBlockArgs._fields_]
    assert pa_lib.pa_block_args_size() == C.sizeof(_cabi.PaBlockArgs)


def _args(**over):
    """Arguments of a call that the host checks accept (the addresses are never followed)."""
    a = _cabi.PaBlockArgs()
    a.struct_size = C.sizeof(a)
    for n in ("output", "query", "key_cache", "value_cache", "key_scale", "value_scale", "context_lens", "block_tables", "bounds"):
        setattr(a, n, 0x10000)
    a.num_seqs, a.num_kv_heads, a.group_size, a.q_len, a.head_size, a.block_size = 4, 8, 8, 1, 128, 16
    a.num_blocks, a.table_width, a.max_context_len = 1000, 256, 4096
    a.kv_dtype, a.kv_quant_mode = _cabi.PA_DTYPE_FP8_E4M3FN, _cabi.PA_QUANT_PER_BLOCK
    a.stride_q_h = a.stride_out_h = 128
    a.stride_q_s = a.stride_out_s = 64 * 128
    a.stride_k_c, a.stride_k_h, a.stride_k_b = 256, 2048, 16384
    a.stride_v_2, a.stride_v_h, a.stride_v_b = 16, 2048, 16384
    a.stride_bt_s = 256
    a.stride_bounds_h, a.stride_bounds_b = 256, 2048
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code", [
    (dict(struct_size=8), -2), (dict(reserved0=1), -4), (dict(reserved1=1), -4), (dict(output=None), -1), (dict(query=None), -1),
    (dict(key_cache=None), -1), (dict(value_cache=None), -1), (dict(key_scale=None), -1), (dict(value_scale=None), -1),
    (dict(context_lens=None), -1), (dict(block_tables=None), -1), (dict(selected_counts=0x1000), -1),
    (dict(num_seqs=0), -4), (dict(num_kv_heads=0), -4), (dict(num_blocks=0), -4), (dict(table_width=0), -4), (dict(max_context_len=-1), -4),
    (dict(group_size=0), -4), (dict(q_len=0), -4), (dict(group_size=65), -3), (dict(group_size=33, q_len=2), -3),
    (dict(head_size=96), -3), (dict(block_size=32), -3), (dict(kv_dtype=7), -3), (dict(kv_quant_mode=3), -3), (dict(kv_quant_mode=-2), -3),
    (dict(kv_dtype=0), -3), (dict(v_transposed=2), -4), (dict(stride_k_b=8), -4), (dict(stride_v_2=24), -4), (dict(key_cache=0x10008), -4),
    (dict(query=0x10008), -4), (dict(stride_q_h=132), -4), (dict(output=0x10004), -4), (dict(stride_out_h=130), -4),
    (dict(selected_blocks=0x1000, num_selected=0), -4), (dict(selected_blocks=0x1000, num_selected=1 << 27), -4),
    (dict(table_width=1 << 27), -4), (dict(max_context_len=(1 << 30) + 1), -4), (dict(num_seqs=1 << 27), -4),
    (dict(kv_quant_mode=1, stride_kvscale_b=3), -4),
])
def test_c_abi_refuses(pa_lib, over, code):
    a = _args(**over)
    assert pa_lib.pa_block_attention_workspace_bytes(C.byref(a)) == code
    assert pa_lib.pa_block_attention(C.byref(a), None) == code


def test_c_abi_refuses_the_other_entry_points(pa_lib):
    for fn in (pa_lib.pa_block_attention, pa_lib.pa_block_bounds, pa_lib.pa_select_blocks):
        assert fn(None, None) == -1
    for over, code in ((dict(bounds=None), -1), (dict(new_tokens=-1), -4), (dict(bounds=0x10004), -4), (dict(stride_bounds_h=12), -4), (dict(key_scale=None), -1)):
        assert pa_lib.pa_block_bounds(C.byref(_args(**over)), None) == code
    ok = dict(selected_blocks=0x20000, selected_counts=0x30000, num_selected=8, recent_blocks=1)
    assert pa_lib.pa_select_blocks_workspace_bytes(C.byref(_args(**ok))) > 0
    assert pa_lib.pa_select_blocks(C.byref(_args(**ok)), None) == -1  # no workspace
    assert pa_lib.pa_select_blocks(C.byref(_args(**ok, workspace=0x40000, workspace_bytes=16)), None) == -7
    for over, code in ((dict(bounds=None), -1), (dict(selected_counts=None), -1), (dict(selected_blocks=None), -1), (dict(num_selected=0), -4),
                       (dict(first_blocks=8), -4), (dict(recent_blocks=9), -4), (dict(first_blocks=-1), -4), (dict(query=None), -1)):
        assert pa_lib.pa_select_blocks_workspace_bytes(C.byref(_args(**{**ok, **over}))) == code
    w = _cabi.PaKvWriteArgs()
    assert pa_lib.pa_kv_cache_write_block_scaled(None, 4, None) == -1
    assert pa_lib.pa_kv_cache_write_block_scaled(C.byref(w), 4, None) == -2
    w.struct_size, w.num_tokens = C.sizeof(w), 3
    assert pa_lib.pa_kv_cache_write_block_scaled(C.byref(w), 4, None) == -1
    for n in ("key", "value", "slot_mapping", "key_cache", "value_cache", "key_scale", "value_scale"):
        setattr(w, n, 0x1000)
    w.num_kv_heads, w.head_size, w.block_size, w.cache_dtype, w.kv_quant_mode = 2, 128, 16, 1, 2
    for over, code in ((dict(num_tokens=-1), -4), (dict(num_tokens=1 << 30), -4), (dict(num_kv_heads=0), -4), (dict(cache_dtype=0), -3), (dict(kv_quant_mode=1), -3),
                       (dict(head_size=96), -3), (dict(block_size=48), -3), (dict(v_transposed=2), -4), (dict(stride_kc_b=8), -4), (dict(key_cache=0x1008), -4)):
        saved = {k: getattr(w, k) for k in over}
        for k, v in over.items():
            setattr(w, k, v)
        assert pa_lib.pa_kv_cache_write_block_scaled(C.byref(w), 4, None) == code, over
        for k, v in saved.items():
            setattr(w, k, v)
    assert pa_lib.pa_kv_cache_write_block_scaled(C.byref(w), 0, None) == -4


def test_existing_entry_points_still_refuse_block_scales(pa_lib):
    """paged_attention_decode and the token-scaled writer know no scale per block."""
    a = _attention()
    with pytest.raises(ValueError, match="Expected key_scale shape"):
        T.plan_decode(a["output"], a["query"], a["key_cache"], a["value_cache"], a["sequence_lengths"], a["block_tables"], 0.1, 1, 40, None, None,
                      a["key_scale"], a["value_scale"])


@pytest.mark.parametrize("mode", [2, 3, 7, -2, 1 << 20])
def test_the_token_scaled_writer_refuses_other_modes(pa_lib, mode):
    """pa_kv_cache_write knows no scale, one scale and one per token; with any other mode it would store codes that no scale
    belongs to.  (No tokens: nothing could be launched, whatever the checks let through.)"""
    w = _cabi.PaKvWriteArgs()
    w.struct_size, w.num_tokens = C.sizeof(w), 0
    for n in ("key", "value", "slot_mapping", "key_cache", "value_cache", "key_scale", "value_scale"):
        setattr(w, n, 0x1000)
    w.num_kv_heads, w.head_size, w.block_size, w.cache_dtype, w.kv_quant_mode = 2, 128, 16, _cabi.PA_DTYPE_FP8_E4M3FN, mode
    assert pa_lib.pa_kv_cache_write(C.byref(w), None) == -3
    for known in (_cabi.PA_QUANT_NONE, _cabi.PA_QUANT_PER_TENSOR, _cabi.PA_QUANT_PER_TOKEN):
        w.kv_quant_mode = known
        assert pa_lib.pa_kv_cache_write(C.byref(w), None) == 0


# ---- the oracle ---------------------------------------------------------------------------------------------------------
def test_oracle_attention_is_torchs():
    g = torch.Generator().manual_seed(0)
    k = torch.randn(6, 2, 16, 64, generator=g).to(torch.bfloat16)
    v = torch.randn(6, 2, 16, 64, generator=g).to(torch.bfloat16)
    kc, vc = k.view(6, 2, 16, 8, 8).permute(0, 1, 3, 2, 4), v.transpose(2, 3)
    q = torch.randn(1, 2 * 3 * 2, 64, generator=g).to(torch.bfloat16)
    table = torch.tensor([[4, 1, 3]], dtype=torch.int32)
    out, lse, _ = O.attention(q, kc, vc, [41], table, 0.125, 2)
    kk = k[[4, 1, 3]].permute(1, 0, 2, 3).reshape(2, 48, 64)[:, :41].double()
    vv = v[[4, 1, 3]].permute(1, 0, 2, 3).reshape(2, 48, 64)[:, :41].double()
    for h in range(2):
        for t in range(2):
            rows = q[0, h * 6 + t * 3:h * 6 + t * 3 + 3].double()
            want = torch.nn.functional.scaled_dot_product_attention(rows[None], kk[None, h, : 40 + t], vv[None, h, : 40 + t], scale=0.125)[0]
            torch.testing.assert_close(out[0, h * 6 + t * 3:h * 6 + t * 3 + 3], want)
    sel = torch.tensor([[[2, 0], [1, 2]]], dtype=torch.int32)
    part, plse, _ = O.attention(q, kc, vc, [41], table, 0.125, 2, selected=sel)
    at = list(range(32, 41)) + list(range(16))
    want = torch.softmax(q[0, 3:6].double() @ kk[0, at].T * 0.125, 1) @ vv[0, at]
    torch.testing.assert_close(part[0, 3:6], want)


def test_oracle_scale_is_the_smallest_power_of_two():
    for bits in list(range(1, 0x7f80, 37)) + [0x7f7f]:
        x = float(torch.tensor(bits, dtype=torch.int16).view(torch.bfloat16))
        s = O.block_scale(x)
        assert math.frexp(s)[0] == 0.5 and x <= 448 * s and (s == 2.0**-126 or x > 448 * s / 2)


def test_oracle_write_moves_codes_by_their_exponent():
    """A scale that grows by powers of two moves codes exactly, but for those that become subnormal."""
    g = torch.Generator().manual_seed(1)
    kc, vc = torch.zeros(1, 1, 4, 16, 16).to(FP8), torch.zeros(1, 1, 64, 16).to(FP8)
    ks, vs = torch.zeros(1, 1, 1, 1), torch.zeros(1, 1, 1, 1)
    small = torch.randn(3, 1, 64, generator=g).to(torch.bfloat16)
    O.write(small, small, kc, vc, torch.tensor([0, 1, 2]), ks, vs)
    before, s0 = kc.double()[0, 0].permute(1, 0, 2).flatten(1)[:3] * float(ks), float(ks)
    O.write(16 * small[:1], small[:1], kc, vc, torch.tensor([9]), ks, vs)
    after = kc.double()[0, 0].permute(1, 0, 2).flatten(1)[:3] * float(ks)
    normal = before.abs() >= 2.0**-6 * float(ks)
    assert float(ks) > s0 and float(vs) == s0 and torch.equal(before[normal], after[normal])
    assert bool(((before - after).abs() <= 2.0**-10 * float(ks)).all())
