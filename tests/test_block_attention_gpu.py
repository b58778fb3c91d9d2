"""The block-granular operators on the GPU against their 64-bit oracle: attention over a cache with one scale per
(block, head), attention over selected blocks, block bounds, block selection, the block-scaled cache write, and the decode
step they make up together.  Tolerances are the oracle's (attention_tolerance: derived from the widths the kernel carries)
plus half a bf16 step of the result; codes, scales, bounds and selections have to be equal."""
import math

import pytest
import torch

from oracle import block_oracle as O

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def _scale(x):
    m, e = torch.frexp(x.abs().amax((2, 3), keepdim=True))
    return torch.ldexp(torch.ones_like(m), torch.where(m <= 0.875, e - 9, e - 8))


def make_cache(g, nblk, hkv, d, bs, mode, vt=False):
    """(key_cache, value_cache, key_scale, value_scale) on the CPU; mode: block, odd (block scales that are no powers of
    two), token, tensor, none (FP8 without scales), bf16."""
    out = []
    for is_key in (True, False):
        x = torch.randn(nblk, hkv, bs, d, generator=g) * torch.exp(0.5 * torch.randn(nblk, hkv, 1, 1, generator=g))
        if mode == "bf16":
            c, s = x.to(torch.bfloat16), None
        else:
            if mode == "block":
                s = _scale(x)
            elif mode == "odd":
                s = x.abs().amax((2, 3), keepdim=True) / 448
            elif mode == "token":
                s = x.abs().amax(3, keepdim=True) / 448
            else:
                s = x.abs().max() / 448 if mode == "tensor" else None
            c = (x / s if s is not None else x).clamp(-448, 448).to(FP8)
        e = 16 // c.element_size()
        if is_key:
            c = c.view(nblk, hkv, bs, d // e, e).permute(0, 1, 3, 2, 4).contiguous()
        elif vt:
            c = c.view(nblk, hkv, bs // e, e, d).permute(0, 1, 2, 4, 3).contiguous()
        else:
            c = c.transpose(2, 3).contiguous()
        out.append((c, s))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def make_table(g, lens, bs, nblk, width=None):
    need = [-(-int(n) // bs) for n in lens]
    perm = torch.randperm(nblk, generator=g).to(torch.int32)
    width = width or max(max(need), 1)
    table = torch.full((len(lens), width), int(perm[0]), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    assert at <= nblk
    return table


def check(cuda, query, kc, vc, lens, table, q_len, ks, vs, selected=None, counts=None, q_lens=None, max_len=None, gpu=None, poison=True):
    """Runs the call and holds output and lse against the oracle; `gpu` replaces tensors of the call by name."""
    import triton_op_amd as T

    d = query.shape[2]
    max_len = int(max(lens.tolist() + [0])) if max_len is None else max_len
    dev = {n: (t.to(cuda) if isinstance(t, torch.Tensor) else t) for n, t in dict(
        query=query, kc=kc, vc=vc, lens=lens, table=table, ks=ks, vs=vs, selected=selected, counts=counts, q_lens=q_lens).items()}
    dev["out"] = torch.full(query.shape, float("nan"), dtype=torch.bfloat16, device=cuda)
    dev["lse"] = torch.full(query.shape[:2], float("nan"), device=cuda)
    dev.update(gpu or {})
    got = T.paged_block_attention(dev["out"], dev["query"], dev["kc"], dev["vc"], dev["lens"], dev["table"], d ** -0.5, q_len, max_len,
                                  dev["ks"], dev["vs"], selected_blocks=dev["selected"], selected_counts=dev["counts"],
                                  query_lens=dev["q_lens"], lse=dev["lse"])
    assert got is dev["out"]
    torch.cuda.synchronize()
    ref, lse, size = O.attention(query, kc, vc, lens, table, d ** -0.5, q_len, ks, vs, selected, counts, q_lens, max_len)
    compare(dev["out"].cpu(), dev["lse"].cpu(), ref, lse, size, kc, vc, vs, table, min(max_len, table.shape[1] * kc.shape[3]), d)
    return dev["out"]


def compare(out, got_lse, ref, lse, size, kc, vc, vs, table, tokens, d):
    v = O.value_tokens(vc)
    v_max = float(torch.nan_to_num(v * vs.double() if vs is not None else v).abs().max())
    p_tol, lse_tol = O.attention_tolerance(lse, size, tokens, d, v_max)
    err = (out.double() - ref).abs() - 2.0**-8 * ref.abs() - p_tol[..., None]
    assert bool((err <= 0).all()), f"output off by {float(err.max()):.3e} beyond its bound at {torch.nonzero(err > 0)[:3].tolist()}"
    seen = lse > -math.inf
    assert torch.equal(got_lse > -math.inf, seen)
    assert bool(((got_lse.double() - lse).abs()[seen] <= lse_tol[seen]).all())
    assert bool((out[~seen] == 0).all())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("mode", ["block", "odd", "token", "tensor", "none", "bf16"])
@pytest.mark.parametrize("bs,vt", [(16, False), (16, True), (64, False), (1024, True), (1024, False)])
def test_attention_over_every_cache(cuda, d, mode, bs, vt):
    g = torch.Generator().manual_seed(d + bs)
    lens = torch.tensor([0, 1, 15, 16, 17, 63, 64, 65, 300, 1025], dtype=torch.int32)
    nblk = sum(-(-int(n) // bs) for n in lens) + 3
    kc, vc, ks, vs = make_cache(g, nblk, 2, d, bs, mode, vt)
    query = torch.randn(len(lens), 2 * 5, d, generator=g).to(torch.bfloat16)
    check(cuda, query, kc, vc, lens, make_table(g, lens, bs, nblk), 1, ks, vs)


@pytest.mark.parametrize("hkv,group,q_len,ragged", [(1, 1, 1, False), (3, 8, 2, False), (2, 16, 1, False), (2, 5, 4, True), (1, 16, 4, True),
                                                    (1, 12, 4, False), (2, 1, 64, False), (8, 8, 1, False), (1, 64, 1, False)])
@pytest.mark.parametrize("d,mode", [(128, "block"), (64, "bf16"), (256, "block"), (128, "token"), (128, "bf16")])
def test_attention_row_layouts(cuda, hkv, group, q_len, ragged, d, mode):
    g = torch.Generator().manual_seed(group * 100 + q_len)
    lens = torch.tensor([3, 700, 64, 1, 129, 2], dtype=torch.int32)
    nblk = 90
    kc, vc, ks, vs = make_cache(g, nblk, hkv, d, 16, mode)
    query = torch.randn(len(lens), hkv * group * q_len, d, generator=g).to(torch.bfloat16)
    q_lens = torch.tensor([1, q_len, 1, 1, max(1, q_len - 1), 0], dtype=torch.int32) if ragged else None
    check(cuda, query, kc, vc, lens, make_table(g, lens, 16, nblk), q_len, ks, vs, q_lens=q_lens)


@pytest.mark.parametrize("lens", [[5000], [9001, 3], [257, 256, 255, 512, 513], [20000, 1, 0, 4097]])
@pytest.mark.parametrize("bs", [16, 1024])
def test_attention_with_a_cut_axis(cuda, lens, bs):
    """Few sequences: the token axis is cut and the stretches are merged by the second kernel."""
    g = torch.Generator().manual_seed(len(lens))
    lens = torch.tensor(lens, dtype=torch.int32)
    nblk = sum(-(-int(n) // bs) for n in lens) + 1
    kc, vc, ks, vs = make_cache(g, nblk, 2, 128, bs, "block")
    query = (2 * torch.randn(len(lens), 2 * 8 * 2, 128, generator=g)).to(torch.bfloat16)
    check(cuda, query, kc, vc, lens, make_table(g, lens, bs, nblk), 2, ks, vs)


def test_attention_ignores_what_lies_behind_a_context(cuda):
    """NaN codes in the slots behind each context and in blocks nobody owns, scales of unowned blocks NaN, table entries behind
    the last block far outside the cache; contexts cut at max_sequence_length and at the table's width."""
    g = torch.Generator().manual_seed(3)
    for mode in ("block", "token", "bf16"):
        lens = torch.tensor([5, 70, 33, 200], dtype=torch.int32)
        kc, vc, ks, vs = make_cache(g, 40, 2, 128, 16, mode)
        table = make_table(g, lens, 16, 40)
        query = torch.randn(4, 2 * 8, 128, generator=g).to(torch.bfloat16)
        live = torch.zeros(40, 16, dtype=torch.bool)
        for b, n in enumerate(lens.tolist()):
            for i in range(-(-n // 16)):
                live[table[b, i], : max(0, min(16, n - 16 * i))] = True
        kc2, vc2 = kc.clone().float(), vc.clone().float()
        kc2.permute(0, 3, 1, 2, 4)[~live] = math.nan
        vc2.permute(0, 3, 1, 2)[~live] = math.nan
        gpu = dict(kc=kc2.to(kc.dtype).to(cuda), vc=vc2.to(vc.dtype).to(cuda))
        if ks is not None:
            dead = ~live.any(1) if mode == "block" else ~live
            k2, v2 = ks.clone(), vs.clone()
            if mode == "block":
                k2[dead], v2[dead] = math.nan, math.nan
            else:
                k2.squeeze(3).transpose(1, 2)[dead] = math.nan
                v2.squeeze(3).transpose(1, 2)[dead] = math.nan
            gpu.update(ks=k2.to(cuda), vs=v2.to(cuda))
        t2 = table.clone()
        for b, n in enumerate(lens.tolist()):
            t2[b, -(-n // 16):] = 2**31 - 1
        gpu["table"] = t2.to(cuda)
        check(cuda, query, kc, vc, lens, table, 1, ks, vs, gpu=gpu)
        check(cuda, query, kc, vc, lens, table, 1, ks, vs, max_len=60)
        check(cuda, query, kc, vc, lens, table[:, :3].contiguous(), 1, ks, vs)


def test_attention_passes_over_bad_blocks(cuda):
    """Entries of the block table outside the cache contribute nothing, wherever they stand."""
    g = torch.Generator().manual_seed(4)
    lens = torch.tensor([100, 64, 16], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, 20, 2, 128, 16, "block")
    table = make_table(g, lens, 16, 20)
    table[0, 2], table[0, 6], table[1, 0], table[2, 0] = -1, 20, -2**31, 2**31 - 1
    query = torch.randn(3, 2 * 4, 128, generator=g).to(torch.bfloat16)
    check(cuda, query, kc, vc, lens, table, 1, ks, vs)


def test_attention_of_strided_tensors(cuda):
    """Blocks inside a larger allocation, heads in another order, query / output / lse rows and table rows with gaps, scales that are
    a slice of something larger."""
    g = torch.Generator().manual_seed(5)
    lens = torch.tensor([100, 333, 18], dtype=torch.int32)
    nblk, hkv, d, bs = 36, 3, 128, 16
    kc, vc, ks, vs = make_cache(g, nblk, hkv, d, bs, "block")
    table = make_table(g, lens, bs, nblk)
    query = torch.randn(3, hkv * 8, d, generator=g).to(torch.bfloat16)

    def inside(t, shape, index):
        big = torch.full(shape, float("nan") if t.dtype != torch.int32 else -7, device=cuda, dtype=torch.float32 if t.dtype == FP8 else t.dtype)
        big = big.to(t.dtype)
        view = big[index]
        view.copy_(t.to(cuda))
        return view

    kbig = torch.zeros(hkv, nblk, d // 16 + 2, bs, 16, dtype=torch.uint8, device=cuda).view(FP8)
    kv = kbig.permute(1, 0, 2, 3, 4)[:, :, : d // 16]
    kv.copy_(kc.to(cuda))
    vbig = torch.zeros(nblk, 2, hkv, d, bs + 16, dtype=torch.uint8, device=cuda).view(FP8)
    vv = vbig[:, 1, :, :, :bs]
    vv.copy_(vc.to(cuda))
    sk = torch.full((nblk, 2, hkv, 1, 1), math.nan, device=cuda)
    sk[:, 0], sk[:, 1] = ks.to(cuda), vs.to(cuda)
    gpu = dict(kc=kv, vc=vv, ks=sk[:, 0], vs=sk[:, 1], table=inside(table, (3, table.shape[1] + 5), (slice(None), slice(0, table.shape[1]))),
               query=inside(query, (5, hkv * 8, 2, d), (slice(1, 4), slice(None), 1)),
               out=inside(torch.zeros_like(query), (3, hkv * 8 + 2, d + 8), (slice(None), slice(1, hkv * 8 + 1), slice(0, d))),
               lse=torch.full((3, 2 * hkv * 8), math.nan, device=cuda)[:, : hkv * 8])
    check(cuda, query, kc, vc, lens, table, 1, ks, vs, gpu=gpu)
    rest = gpu["out"]._base if gpu["out"]._base is not None else gpu["out"]
    assert bool(rest[:, 0].isnan().all()) and bool(rest[:, :, d:].isnan().all())  # nothing beside the rows was written


def test_one_of_everything_with_strides_that_mean_nothing(cuda):
    """One sequence, head, row and block: the strides of those dimensions may be any number, in each of the operators."""
    import triton_op_amd as T

    def odd(t, *dims):
        return t.as_strided(t.shape, [7 if i in dims else st for i, st in enumerate(t.stride())])

    g = torch.Generator().manual_seed(23)
    lens, table = torch.tensor([13], dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    query = torch.randn(1, 1, 128, generator=g).to(torch.bfloat16)
    for mode in ("block", "token"):
        kc, vc, ks, vs = make_cache(g, 1, 1, 128, 16, mode, True)
        one = (0, 1, 2) if mode == "block" else (0, 1)
        check(cuda, query, kc, vc, lens, table, 1, ks, vs, gpu=dict(
            query=odd(query.to(cuda), 0, 1), kc=odd(kc.to(cuda), 0, 1), vc=odd(vc.to(cuda), 0, 1, 2), ks=odd(ks.to(cuda), *one), vs=odd(vs.to(cuda), *one),
            out=odd(torch.zeros(1, 1, 128, dtype=torch.bfloat16, device=cuda), 0, 1), lse=odd(torch.zeros(1, 1, device=cuda), 0, 1),
            table=odd(table.to(cuda), 0, 1)))
        want = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
        box = odd(want.to(cuda), 0, 1)
        T.key_block_bounds(box, odd(kc.to(cuda), 0, 1), lens.to(cuda), odd(table.to(cuda), 0, 1), 13, odd(ks.to(cuda), *one))
        O.bounds(want, kc, lens, table, ks)
        assert torch.equal(box.cpu(), want)
        sel, cnt = T.select_blocks(odd(query.to(cuda), 0, 1), box, lens.to(cuda), table.to(cuda), 1, 16, 1, 13)
        assert sel.tolist() == [[[0]]] and cnt.tolist() == [[1]]
    key, value = _rows(g, 5, 1, 128)
    host = [torch.zeros(1, 1, 8, 16, 16).to(FP8), torch.zeros(1, 1, 1, 128, 16).to(FP8), torch.zeros(1, 1, 1, 1), torch.zeros(1, 1, 1, 1)]
    dev = [odd(t.to(cuda), *dims) for t, dims in zip(host, ((0, 1), (0, 1), (0, 1, 2), (0, 1)))]
    T.kv_cache_write(key.to(cuda), value.to(cuda), dev[0], dev[1], torch.arange(5, device=cuda), dev[2], dev[3])
    O.write(key, value, *host[:2], torch.arange(5), *host[2:])
    for a, b in zip(dev, host):
        assert torch.equal(a.cpu().float(), b.float())


def test_attention_in_a_cache_beyond_32_bit_offsets(cuda):
    """Blocks at both ends of a cache of more than 2^32 bytes."""
    g = torch.Generator().manual_seed(6)
    hkv, d, bs, nblk = 8, 128, 16, 270000  # 4.4e9 bytes of keys, as many of values
    lens = torch.tensor([90, 40], dtype=torch.int32)
    small = make_cache(g, 9, hkv, d, bs, "block")
    where = torch.tensor([0, nblk - 1, 131072, 262144, 269000, 1, 200000, 262143, 131071])
    big = [torch.empty((nblk,) + tuple(t.shape[1:]), dtype=t.dtype, device=cuda) for t in small]
    for t, s in zip(big, small):
        t[where.to(cuda)] = s.to(cuda)
    order = torch.arange(9, dtype=torch.int32)
    table = torch.full((2, 6), 0, dtype=torch.int32)
    table[0], table[1, :3] = order[:6], order[6:]
    query = torch.randn(2, hkv * 8, d, generator=g).to(torch.bfloat16)
    gpu = dict(kc=big[0], vc=big[1], ks=big[2], vs=big[3], table=where.to(torch.int32)[table.long()].to(cuda))
    check(cuda, query, small[0], small[1], lens, table, 1, small[2], small[3], gpu=gpu)


@pytest.mark.parametrize("scale", [0.0, 30.0, -1.0])
def test_attention_softmax_extremes(cuda, scale):
    """Equal logits, logits of some thousands in both directions, a negative softmax scale."""
    import triton_op_amd as T

    g = torch.Generator().manual_seed(8)
    lens = torch.tensor([700, 40], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, 50, 1, 128, 16, "block")
    table = make_table(g, lens, 16, 50)
    query = torch.randn(2, 8, 128, generator=g).to(torch.bfloat16)
    out, lse = torch.empty_like(query, device=cuda), torch.empty(2, 8, device=cuda)
    T.paged_block_attention(out, query.to(cuda), kc.to(cuda), vc.to(cuda), lens.to(cuda), table.to(cuda), scale, 1, 700, ks.to(cuda), vs.to(cuda), lse=lse)
    ref, rlse, size = O.attention(query, kc, vc, lens, table, scale, 1, ks, vs)
    compare(out.cpu(), lse.cpu(), ref, rlse, size, kc, vc, vs, table, 700, 128)


def _with_signs(g, s):
    return s * (2.0 * torch.randint(0, 2, s.shape, generator=g) - 1)


@pytest.mark.parametrize("d,group,q_len,bs,vt", [(128, 8, 1, 16, False), (128, 16, 4, 16, False), (128, 5, 2, 1024, True), (64, 8, 1, 64, False),
                                                 (64, 12, 3, 16, True), (256, 8, 1, 16, False), (256, 16, 2, 64, False)])
@pytest.mark.parametrize("mode", ["block", "odd"])
def test_attention_with_block_scales_of_either_sign(cuda, d, group, q_len, bs, vt, mode):
    """Block scales below zero among the others, -0.0 and subnormal ones: a key or value is code * scale, whatever its sign.  The
    queries are large enough that a softmax reference taken from the wrong end overflows."""
    g = torch.Generator().manual_seed(d + group)
    lens = torch.tensor([700, 64, 1, 2049, 17], dtype=torch.int32)
    nblk = sum(-(-int(n) // bs) for n in lens) + 2
    kc, vc, ks, vs = make_cache(g, nblk, 2, d, bs, mode, vt)
    ks, vs = _with_signs(g, ks), _with_signs(g, vs)
    table = make_table(g, lens, bs, nblk)
    ks[table[0, 0], 0], vs[table[3, 1], 0] = -0.0, -0.0
    vs[table[3, 2], 0], vs[table[0, 1] if bs < 1024 else table[1, 0], 1] = 2.0**-130, -(2.0**-131) * 1.5
    query = torch.randn(len(lens), 2 * group * q_len, d, generator=g)
    for size, k, v in ((4, ks, vs), (40, ks, vs), (40, -ks.abs(), -vs.abs())):
        check(cuda, (size * query).to(torch.bfloat16), kc, vc, lens, table, q_len, k, v)


# ---- selected blocks ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d,mode,bs,vt", [(128, "block", 16, False), (128, "bf16", 16, True), (64, "token", 64, False), (256, "block", 64, True),
                                          (128, "tensor", 1024, False)])
@pytest.mark.parametrize("group,q_len,ragged", [(8, 1, False), (6, 3, True), (16, 4, False)])
def test_attention_over_selected_blocks(cuda, d, mode, bs, vt, group, q_len, ragged):
    """Lists in any order, with numbers outside the sequence among them, counts below and at the list's length."""
    g = torch.Generator().manual_seed(d + group)
    lens = torch.tensor([40 * bs + 3, 0, 5, 7 * bs, 12 * bs - 1], dtype=torch.int32)
    nblk, hkv, k = 70, 2, 9
    kc, vc, ks, vs = make_cache(g, nblk, hkv, d, bs, mode, vt)
    table = make_table(g, lens, bs, nblk)
    query = torch.randn(len(lens), hkv * group * q_len, d, generator=g).to(torch.bfloat16)
    selected = torch.empty(len(lens), hkv, k, dtype=torch.int32)
    for b, n in enumerate(lens.tolist()):
        blocks = -(-n // bs)
        for h in range(hkv):
            order = torch.randperm(max(blocks, k) + 3, generator=g)[:k].to(torch.int32)
            order[int(torch.randint(0, k, (1,), generator=g))] = [-1, 2**31 - 1][h]
            selected[b, h] = order
    counts = torch.tensor([[k, 4], [k, 0], [1, k], [0, k], [k + 5, 3]], dtype=torch.int32)
    q_lens = torch.tensor([1, q_len, 2, q_len, 1], dtype=torch.int32) if ragged else None
    for c in (counts, None):
        check(cuda, query, kc, vc, lens, table, q_len, ks, vs, selected, c, q_lens)


def test_attention_over_all_blocks_as_a_list_is_the_dense_call(cuda):
    g = torch.Generator().manual_seed(9)
    lens = torch.tensor([333, 1200], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, 100, 2, 128, 16, "block")
    table = make_table(g, lens, 16, 100)
    query = torch.randn(2, 16, 128, generator=g).to(torch.bfloat16)
    every = torch.arange(table.shape[1], dtype=torch.int32).expand(2, 2, -1).contiguous()
    dense = check(cuda, query, kc, vc, lens, table, 1, ks, vs)
    listed = check(cuda, query, kc, vc, lens, table, 1, ks, vs, every)
    torch.testing.assert_close(dense.float(), listed.float(), atol=0, rtol=2.0**-7)  # (one step of bf16: other stretches)


# ---- bounds -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("mode", ["block", "odd", "token", "tensor", "none", "bf16"])
@pytest.mark.parametrize("bs", [16, 64, 1024])
def test_bounds(cuda, d, mode, bs):
    import triton_op_amd as T

    g = torch.Generator().manual_seed(d + bs)
    lens = torch.tensor([0, 1, bs, bs + 1, 4 * bs - 1, 130], dtype=torch.int32)
    nblk = 24
    kc, _, ks, _ = make_cache(g, nblk, 3, d, bs, mode)
    kf = kc.float()
    kf[:, 1, 0, 0, 3] = math.nan  # a NaN among the keys is passed over
    kf[:, 2, 0, :, 0] = math.nan  # a head dim with nothing else is left without bounds
    kc = kf.to(kc.dtype)
    table = make_table(g, lens, bs, nblk)
    table[5, -1] = 77 if table.shape[1] > -(-130 // bs) else table[5, -1]
    for new in (None, 1, 3, 4 * bs):
        got = torch.full((nblk, 3, 2, d), 5.0, dtype=torch.bfloat16)
        want, dev = got.clone(), got.to(cuda)
        for n in (lens, lens):
            assert T.key_block_bounds(dev, kc.to(cuda), n.to(cuda), table.to(cuda), int(n.max()), ks.to(cuda) if ks is not None else None, new_tokens=new) is dev
        O.bounds(want, kc, lens, table, ks, new)
        torch.cuda.synchronize()
        assert torch.equal(dev.cpu().view(torch.int16) & 0x7fff, want.view(torch.int16) & 0x7fff) and torch.equal(dev.cpu(), want)


@pytest.mark.parametrize("mode", ["block", "tensor", "token"])
@pytest.mark.parametrize("bs", [16, 64])
def test_bounds_with_scales_of_either_sign_and_zero(cuda, mode, bs):
    """A negative scale turns the smallest code into the largest key; a head dim without a number has no bounds (+infinity,
    -infinity) whatever the scale is, zero too."""
    import triton_op_amd as T

    g = torch.Generator().manual_seed(bs)
    lens = torch.tensor([5 * bs - 3, 1, bs], dtype=torch.int32)
    kc, _, ks, _ = make_cache(g, 8, 3, 128, bs, mode)
    kf = kc.float()
    kf[:, 1, 0, :, 3], kf[:, 2, 3, :, 0] = math.nan, math.nan
    kc = kf.to(kc.dtype)
    table = make_table(g, lens, bs, 8)
    signed = [_with_signs(g, ks), -ks.abs(), torch.zeros_like(ks), -torch.zeros_like(ks)]
    if ks.dim():
        signed.append(_with_signs(g, ks) * torch.randint(0, 2, ks.shape, generator=g))
    for s in signed:
        want = torch.full((8, 3, 2, 128), 5.0, dtype=torch.bfloat16)
        dev = want.to(cuda)
        T.key_block_bounds(dev, kc.to(cuda), lens.to(cuda), table.to(cuda), int(lens.max()), s.to(cuda))
        O.bounds(want, kc, lens, table, s)
        torch.cuda.synchronize()
        assert torch.equal(dev.cpu(), want)


def test_bounds_of_strided_tensors_and_bad_entries(cuda):
    import triton_op_amd as T

    g = torch.Generator().manual_seed(2)
    lens = torch.tensor([70, 33], dtype=torch.int32)
    kc, _, ks, _ = make_cache(g, 12, 2, 128, 16, "block")
    table = make_table(g, lens, 16, 12, width=6)
    table[0, 1], table[1, 0], table[0, 5] = 12, -3, 2**30
    big = torch.full((12, 4, 2, 128), 3.0, dtype=torch.bfloat16, device=cuda)
    want = torch.full((12, 2, 2, 128), 3.0, dtype=torch.bfloat16)
    kb = torch.zeros(12, 4, 8, 16, 16, dtype=torch.uint8, device=cuda).view(FP8)
    kb[:, 1:3] = kc.to(cuda)
    T.key_block_bounds(big[:, 1:3], kb[:, 1:3], lens.to(cuda), table.to(cuda), 70, ks.to(cuda))
    O.bounds(want, kc, lens, table, ks)
    torch.cuda.synchronize()
    assert torch.equal(big[:, 1:3].cpu(), want) and bool((big[:, 0] == 3).all()) and bool((big[:, 3] == 3).all())


# ---- selection ---------------------------------------------------------------------------------------------------------------
def _box(g, nblk, hkv, d):
    c, w = torch.randn(nblk, hkv, d, generator=g), torch.randn(nblk, hkv, d, generator=g).abs()
    return torch.stack((c - w, c + w), 2).to(torch.bfloat16)


def check_select(cuda, query, box, lens, table, k, bs, q_len, first=0, recent=None, q_lens=None, max_len=None, **kw):
    import triton_op_amd as T

    need = 1 + -(-(q_len - 1) // bs)
    max_len = int(lens.max()) if max_len is None else max_len
    sel, cnt = T.select_blocks(query.to(cuda), box.to(cuda), lens.to(cuda), table.to(cuda), k, bs, q_len, max_len, first_blocks=first,
                               recent_blocks=recent, query_lens=None if q_lens is None else q_lens.to(cuda), **kw)
    want, counts = O.select(query, box, lens, table, k, bs, q_len, first, need if recent is None else recent, q_lens, max_len)
    torch.cuda.synchronize()
    assert torch.equal(cnt.cpu(), counts)
    assert torch.equal(sel.cpu(), want)
    return sel, cnt


@pytest.mark.parametrize("d,hkv,group,q_len", [(128, 2, 8, 1), (64, 1, 16, 4), (256, 3, 5, 2), (128, 1, 1, 1), (128, 8, 8, 1), (64, 2, 1, 33)])
@pytest.mark.parametrize("bs", [16, 64])
def test_selection(cuda, d, hkv, group, q_len, bs):
    g = torch.Generator().manual_seed(d + q_len)
    lens = torch.tensor([0, 1, bs * 5, bs * 40 + 3, bs * 333 - 1, bs * 12], dtype=torch.int32)
    nblk = 400
    box, table = _box(g, nblk, hkv, d), make_table(g, lens, bs, nblk)
    query = torch.randn(len(lens), hkv * group * q_len, d, generator=g).to(torch.bfloat16)
    q_lens = torch.tensor([1, 1, q_len, max(1, q_len - 1), q_len, 1], dtype=torch.int32) if q_len > 1 else None
    for k, first, recent in ((12, 0, None), (12, 2, 6), (1 + -(-(q_len - 1) // bs), 0, None), (400, 1, 5), (40, 0, 40)):
        check_select(cuda, query, box, lens, table, k, bs, q_len, first, recent, q_lens)
    check_select(cuda, query, box, lens, table, 9, bs, q_len, 1, None, None, max_len=bs * 30)
    check_select(cuda, query, box, lens, table[:, :20].contiguous(), 9, bs, q_len, 1)


def test_selection_ties_go_to_the_lower_block(cuda):
    g = torch.Generator().manual_seed(1)
    lens = torch.tensor([16 * 3000, 16 * 1500 + 5], dtype=torch.int32)
    box = _box(g, 7, 2, 128)  # seven different boxes for 3000 blocks
    table = torch.randint(0, 7, (2, 3000), generator=g).to(torch.int32)
    query = torch.randn(2, 16, 128, generator=g).to(torch.bfloat16)
    for k in (1, 10, 1000, 2999):
        check_select(cuda, query, box, lens, table, k, 16, 1)
    check_select(cuda, torch.zeros_like(query), box, lens, table, 100, 16, 1, 3, 2)  # every score is zero, of either sign


def test_selection_of_scores_that_differ_in_the_last_bits_of_32(cuda):
    """Scores whose difference is far below a 32-bit rounding of their sums: only an exact sum ranks them."""
    n, d = 600, 128
    box = torch.zeros(n, 1, 2, d)
    box[:, 0, :, 0] = 256.0          # q = 1: every score has 256 - 256 + something tiny in it, in different places
    box[:, 0, :, 127] = -256.0
    tiny = torch.randperm(n, generator=torch.Generator().manual_seed(0)).float() * 2.0**-30
    hi = tiny.to(torch.bfloat16).float()
    box[:, 0, :, 64], box[:, 0, :, 65] = hi[:, None], (tiny - hi).to(torch.bfloat16).float()[:, None]
    box = box.to(torch.bfloat16)
    query = torch.ones(1, 1, d, dtype=torch.bfloat16)
    lens, table = torch.tensor([16 * n], dtype=torch.int32), torch.arange(n, dtype=torch.int32)[None]
    for k in (5, 77, 300):
        check_select(cuda, query, box, lens, table, k, 16, 1)


def test_selection_with_bounds_that_are_no_numbers(cuda):
    g = torch.Generator().manual_seed(11)
    lens = torch.tensor([16 * 60, 16 * 44], dtype=torch.int32)
    box, table = _box(g, 110, 2, 128), make_table(g, lens, 16, 110)
    box[::7, 0, 1, 5] = math.nan
    box[::5, 1, 1, :] = math.inf
    box[1::9, :, 0, :], box[1::9, :, 1, :] = math.inf, -math.inf  # a block without keys
    box[3::11] = 3.0e38
    table[0, 7], table[1, 3] = -1, 110  # not blocks of the cache: they rank last
    query = torch.randn(2, 2 * 4, 128, generator=g).to(torch.bfloat16)
    query[0, 1] = math.nan
    query[1, 2] = query[1, 2].abs() + 1
    for k in (5, 20, 43, 59):
        check_select(cuda, query, box, lens, table, k, 16, 1, 1, 2)


def test_selection_from_more_blocks_than_the_flags_hold(cuda):
    """More than 65536 blocks (a million tokens in blocks of 16): every score is formed in 64 bits."""
    g = torch.Generator().manual_seed(13)
    n = 65536 + 777
    lens = torch.tensor([16 * n - 5, 16 * 3000], dtype=torch.int32)
    box, table = _box(g, n, 1, 64), torch.stack([torch.randperm(n, generator=g), torch.randint(0, n, (n,), generator=g)]).to(torch.int32)
    table[0, 70] = -1
    query = torch.randn(2, 2, 64, generator=g).to(torch.bfloat16)
    for k, first, recent in ((300, 1, 2), (3, 1, 2), (20000, 0, 1)):
        check_select(cuda, query, box, lens, table, k, 16, 1, first, recent)
    check_select(cuda, torch.cat([query, query], 1), box, lens, table, 9, 16, 2, 1, 3, torch.tensor([0, 1], dtype=torch.int32))


@pytest.mark.parametrize("size", [3.0, 30.0, 100.0, 1.0e6])
@pytest.mark.parametrize("k", [256, 1024, 4096])
def test_selection_with_one_block_of_large_keys(cuda, size, k):
    """The first block's keys are often the largest by far.  They widen the 32-bit stage's intervals and errors, so that many or
    all blocks are left to the 64-bit stage."""
    g = torch.Generator().manual_seed(14)
    n = 8192
    box, table = _box(g, n, 1, 128), torch.randperm(n, generator=g).to(torch.int32)[None]
    box[table[0, 0].long()] *= size
    query = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16)
    check_select(cuda, query, box, torch.tensor([16 * n], dtype=torch.int32), table, k, 16, 1)


def test_selection_of_the_largest_rows(cuda):
    """64 query rows of head size 256: the query operands fill the 64 KiB of LDS that a launch may ask for."""
    g = torch.Generator().manual_seed(15)
    lens = torch.tensor([64 * 150 - 1, 64 * 20, 70], dtype=torch.int32)
    box, table = _box(g, 180, 2, 256), make_table(g, lens, 64, 180)
    query = torch.randn(3, 2 * 64, 256, generator=g).to(torch.bfloat16)
    for q_len in (1, 4):
        check_select(cuda, query, box, lens, table, 17, 64, q_len, 1)


def test_selection_into_the_callers_tensors(cuda):
    g = torch.Generator().manual_seed(12)
    lens = torch.tensor([16 * 30, 100], dtype=torch.int32)
    box, table = _box(g, 40, 2, 64), make_table(g, lens, 16, 40)
    query = torch.randn(2, 8, 64, generator=g).to(torch.bfloat16)
    sel = torch.full((2, 3, 9), 55, dtype=torch.int32, device=cuda)
    cnt = torch.full((2, 5), 55, dtype=torch.int32, device=cuda)
    ws = torch.full((2 * 2 * 30 * 8,), 255, dtype=torch.uint8, device=cuda)
    a, b = check_select(cuda, query, box, lens, table, 8, 16, 1, selected_blocks=sel[:, :2, :8], selected_counts=cnt[:, 1:3], workspace=ws)
    assert a.data_ptr() == sel.data_ptr() and bool((sel[:, 2] == 55).all()) and bool((sel[..., 8] == 55).all())
    assert bool((cnt[:, [0, 3, 4]] == 55).all())


# ---- the write ------------------------------------------------------------------------------------------------------------------
def check_write(cuda, calls, nblk, hkv, d, bs, vt, ks0=None):
    """The same calls on the GPU and on the oracle, from a cache of zeros (or scales `ks0`): equal bytes and scales."""
    import triton_op_amd as T

    kc = torch.zeros(nblk, hkv, d // 16, bs, 16).to(FP8)
    vc = torch.zeros((nblk, hkv, bs // 16, d, 16) if vt else (nblk, hkv, d, bs)).to(FP8)
    ks = torch.zeros(nblk, hkv, 1, 1) if ks0 is None else ks0.clone()
    vs = ks.clone()
    dev = [t.to(cuda) for t in (kc, vc, ks, vs)]
    for key, value, slots in calls:
        T.kv_cache_write(key.to(cuda) if not key.is_cuda else key, value.to(cuda) if not value.is_cuda else value, dev[0], dev[1], slots.to(cuda), dev[2], dev[3])
        O.write(key.cpu(), value.cpu(), kc, vc, slots, ks, vs)
    torch.cuda.synchronize()
    assert torch.equal(dev[2].cpu(), ks) and torch.equal(dev[3].cpu(), vs)
    for got, want in ((dev[0], kc), (dev[1], vc)):
        got, want = got.cpu().float(), want.float()  # (codes as values: a NaN is a NaN)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    return dev


def _rows(g, n, hkv, d, spread=1.5):
    return [(torch.randn(n, hkv, d, generator=g) * torch.exp(spread * torch.randn(n, hkv, 1, generator=g))).to(torch.bfloat16) for _ in range(2)]


@pytest.mark.parametrize("d,hkv,bs,vt", [(128, 2, 16, False), (128, 3, 64, True), (64, 2, 1024, False), (256, 1, 16, True), (256, 2, 64, False), (64, 8, 16, True)])
def test_write_matches_the_oracle_bit_for_bit(cuda, d, hkv, bs, vt):
    """Prompts, continuations, single tokens over blocks that already hold some, tokens that share a slot, padding, slots outside
    the cache: in several calls, so scales grow and codes follow."""
    g = torch.Generator().manual_seed(d + bs)
    nblk = 12 if bs < 1024 else 4
    calls = []
    for n in (1, 3, 17, 64, 200, 1, 2):
        key, value = _rows(g, n, hkv, d)
        slots = torch.randint(0, nblk * bs, (n,), generator=g) if n != 64 else torch.arange(64) + 5
        if n == 200:
            slots[::17] = -1
            slots[1], slots[2], slots[3] = nblk * bs, -5, 2**62
            slots[100:110] = slots[90:100]
        calls.append((key, value, slots))
    check_write(cuda, calls, nblk, hkv, d, bs, vt)


@pytest.mark.parametrize("hkv,bs,vt", [(8, 16, False), (2, 64, True), (1, 1024, False)])
def test_write_of_long_prompts(cuda, hkv, bs, vt):
    """More than 1024 tokens (windows of 16, all heads in a workgroup): runs that end inside blocks, scattered tokens between them,
    and a block that is visited at both ends of the call."""
    g = torch.Generator().manual_seed(bs)
    nblk = 3000 // bs + 4
    order = torch.randperm(nblk, generator=g)
    pos = torch.arange(2500)
    slots = order[pos // bs] * bs + pos % bs
    slots[700:720] = torch.randint(0, nblk * bs, (20,), generator=g)
    slots[-3:] = slots[:3]  # the first block again, by later tokens
    slots[40:45] = -1
    key, value = _rows(g, 2500, hkv, 128)
    k2, v2 = _rows(g, 1100, hkv, 128)
    check_write(cuda, [(key, value, slots), (4 * k2, v2 / 8, slots[300:1400])], nblk, hkv, 128, bs, vt)


def test_write_of_values_that_are_no_numbers(cuda):
    g = torch.Generator().manual_seed(1)
    key, value = _rows(g, 40, 2, 128)
    key[3, 0, 5], key[4, 0, 6], key[5, 1, :], value[6, 1, 7], value[7] = math.inf, math.nan, math.nan, -math.inf, 0.0
    key[20:36] = 0.0
    value[20:36] = 1e-40  # subnormal in bf16: the scale stays at 2^-126
    key[36], key[37] = 3.3e38, 448.0 * 2.0**-20
    slots = torch.arange(40)
    dev = check_write(cuda, [(key, value, slots), (key, value, slots)], 4, 2, 128, 16, False)
    assert bool(dev[0].float().isnan().any()) and bool(dev[2].isfinite().all())


def test_write_keeps_given_scales_that_are_no_powers_of_two(cuda):
    g = torch.Generator().manual_seed(2)
    ks0 = torch.rand(6, 2, 1, 1, generator=g) * 0.01
    calls = [(*_rows(g, n, 2, 128, 2.5), torch.randint(0, 96, (n,), generator=g)) for n in (5, 30, 2, 60)]
    check_write(cuda, calls, 6, 2, 128, 16, False, ks0)


def test_write_of_strided_and_unaligned_rows(cuda):
    import triton_op_amd as T

    g = torch.Generator().manual_seed(3)
    big = torch.randn(50, 2, 3, 131, generator=g).to(torch.bfloat16).to(cuda)
    slots = torch.randperm(96, generator=g)[:50]
    for lo in (0, 1):  # rows at odd element offsets are read element by element
        check_write(cuda, [(big[:, 0, :, lo:lo + 128], big[:, 1, :, lo:lo + 128], slots)], 6, 3, 128, 16, False)
    # cache and scales inside larger allocations: nothing beside them changes
    key, value = (t.to(cuda) for t in _rows(g, 50, 2, 128))
    kb = torch.full((6, 4, 8, 16, 16), 1.0, device=cuda).to(FP8)
    vb = torch.full((6, 4, 128, 16), 1.0, device=cuda).to(FP8)
    sb = torch.full((6, 2, 4, 1, 1), 0.0, device=cuda)
    T.kv_cache_write(key, value, kb[:, 1:3], vb[:, 1:3], slots.to(cuda), sb[:, 0, 1:3], sb[:, 1, 1:3])
    want = [t.cpu() for t in (torch.ones(6, 2, 8, 16, 16).to(FP8), torch.ones(6, 2, 128, 16).to(FP8), torch.zeros(6, 2, 1, 1), torch.zeros(6, 2, 1, 1))]
    O.write(key.cpu(), value.cpu(), want[0], want[1], slots, want[2], want[3])
    torch.cuda.synchronize()
    for got, w in ((kb, want[0]), (vb, want[1])):
        assert torch.equal(got[:, 1:3].cpu().float(), w.float()) and bool((got[:, [0, 3]].float() == 1).all())
    assert torch.equal(sb[:, 0, 1:3].cpu(), want[2]) and torch.equal(sb[:, 1, 1:3].cpu(), want[3]) and bool((sb[:, :, [0, 3]] == 0).all())


def test_write_nothing(cuda):
    import triton_op_amd as T

    kc, vc = torch.zeros(2, 1, 8, 16, 16, device=cuda).to(FP8), torch.zeros(2, 1, 128, 16, device=cuda).to(FP8)
    s = [torch.ones(2, 1, 1, 1, device=cuda) for _ in range(2)]
    none = torch.empty(0, 1, 128, dtype=torch.bfloat16, device=cuda)
    T.kv_cache_write(none, none, kc, vc, torch.empty(0, dtype=torch.int64, device=cuda), *s)
    one = torch.ones(1, 1, 128, dtype=torch.bfloat16, device=cuda)
    T.kv_cache_write(one, one, kc, vc, torch.tensor([-1], device=cuda), *s)
    torch.cuda.synchronize()
    assert float(kc.float().abs().sum()) == 0 and float(s[0].sum()) == 2


# ---- together --------------------------------------------------------------------------------------------------------------------
class _Session:
    """A small serving session: prompts, then decode steps, over one block-scaled cache; the oracle keeps a second cache."""

    def __init__(self, cuda, bs=16, d=128, hkv=2, group=4, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        self.cuda, self.bs, self.d, self.hkv, self.group = cuda, bs, d, hkv, group
        self.lens = torch.tensor([70, 500, 16], dtype=torch.int32)
        self.nblk = 60
        self.table = make_table(self.g, self.lens + 64, bs, self.nblk)
        self.host = [torch.zeros(self.nblk, hkv, d // 16, bs, 16).to(FP8), torch.zeros(self.nblk, hkv, d, bs).to(FP8),
                     torch.zeros(self.nblk, hkv, 1, 1), torch.zeros(self.nblk, hkv, 1, 1),
                     torch.zeros(self.nblk, hkv, 2, d, dtype=torch.bfloat16)]
        self.dev = [t.to(cuda) for t in self.host]

    def slots(self, b, lo, hi):
        pos = torch.arange(lo, hi)
        return self.table[b, pos // self.bs].long() * self.bs + pos % self.bs

    def prompt(self):
        import triton_op_amd as T

        slots = torch.cat([self.slots(b, 0, int(n)) for b, n in enumerate(self.lens)])
        key, value = _rows(self.g, len(slots), self.hkv, self.d, 0.3)
        T.kv_cache_write(key.to(self.cuda), value.to(self.cuda), *self.dev[:2], slots.to(self.cuda), *self.dev[2:4])
        T.key_block_bounds(self.dev[4], self.dev[0], self.lens.to(self.cuda), self.table.to(self.cuda), 500, self.dev[2])
        O.write(key, value, self.host[0], self.host[1], slots, self.host[2], self.host[3])
        O.bounds(self.host[4], self.host[0], self.lens, self.table, self.host[2])

    def step_inputs(self, q):
        key, value = _rows(self.g, 3 * q, self.hkv, self.d, 0.3)
        slots = torch.cat([self.slots(b, int(n), int(n) + q) for b, n in enumerate(self.lens)])
        self.lens = self.lens + q
        query = torch.randn(3, self.hkv * q * self.group, self.d, generator=self.g).to(torch.bfloat16)
        return key, value, slots, self.lens.clone(), query

    def oracle_step(self, q, key, value, slots, lens, query, k):
        O.write(key, value, self.host[0], self.host[1], slots, self.host[2], self.host[3])
        O.bounds(self.host[4], self.host[0], lens, self.table, self.host[2], q)
        sel, cnt = O.select(query, self.host[4], lens, self.table, k, self.bs, q, 1, 2)
        return sel, cnt, O.attention(query, self.host[0], self.host[1], lens, self.table, self.d ** -0.5, q, self.host[2], self.host[3], sel, cnt)

    def gpu_step(self, q, key, value, slots, lens, query, out, lse, k):
        import triton_op_amd as T

        T.kv_cache_write(key, value, *self.dev[:2], slots, *self.dev[2:4])
        T.key_block_bounds(self.dev[4], self.dev[0], lens, self.tbl, 564, self.dev[2], new_tokens=q)
        sel, cnt = T.select_blocks(query, self.dev[4], lens, self.tbl, k, self.bs, q, 564, first_blocks=1, recent_blocks=2)
        T.paged_block_attention(out, query, *self.dev[:2], lens, self.tbl, self.d ** -0.5, q, 564, *self.dev[2:4], selected_blocks=sel,
                                selected_counts=cnt, lse=lse)
        return sel, cnt

    def check_step(self, got, want, out, lse):
        torch.cuda.synchronize()
        assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])
        compare(out.cpu(), lse.cpu(), *want[2], self.host[0], self.host[1], self.host[3], self.table, 564, self.d)
        for a, b in zip(self.dev, self.host):
            assert torch.equal(a.cpu().float(), b.float())


@pytest.mark.parametrize("q", [1, 3])
def test_a_session_step_by_step(cuda, q):
    s = _Session(cuda)
    s.tbl = s.table.to(cuda)
    s.prompt()
    for _ in range(6):
        x = s.step_inputs(q)
        out = torch.empty_like(x[4], device=cuda)
        lse = torch.empty(out.shape[:2], device=cuda)
        got = s.gpu_step(q, *(t.to(cuda) for t in x), out, lse, 12)
        s.check_step(got, s.oracle_step(q, *x, 12), out, lse)


def test_a_session_captured_and_replayed(cuda):
    """The whole step captured once into a graph and replayed with new inputs, with eager work of the program between the
    replays; every replay is held against the oracle."""
    s = _Session(cuda, seed=5)
    s.tbl = s.table.to(cuda)
    s.prompt()
    x = s.step_inputs(1)
    fixed = [t.to(cuda) for t in x]
    out = torch.empty_like(fixed[4])
    lse = torch.empty(out.shape[:2], device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = s.gpu_step(1, *fixed, out, lse, 12)  # the eager first step, on another stream than the tensors' own
    torch.cuda.current_stream().wait_stream(side)
    s.check_step(got, s.oracle_step(1, *x, 12), out, lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = s.gpu_step(1, *fixed, out, lse, 12)
    for i in range(4):
        x = s.step_inputs(1)
        for f, t in zip(fixed, x):
            f.copy_(t)
        out.fill_(math.nan)
        junk = torch.randn(1000, 1000, device=cuda) @ torch.randn(1000, 1000, device=cuda)
        if i % 2:
            torch.cuda.synchronize()
        graph.replay()
        junk.sum().item()
        s.check_step(got, s.oracle_step(1, *x, 12), out, lse)


def test_plans_replay_and_keep_apart(cuda):
    """Two plans on two streams, each with its own workspace, replayed in turn."""
    import triton_op_amd as T

    g = torch.Generator().manual_seed(7)
    lens = torch.tensor([3000], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, 200, 2, 128, 16, "block")
    table = make_table(g, lens, 16, 200)
    plans, refs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    dev = [t.to(cuda) for t in (kc, vc, lens, table, ks, vs)]
    for i in range(2):
        query = torch.randn(1, 16, 128, generator=g).to(torch.bfloat16)
        out, lse = torch.empty(1, 16, 128, dtype=torch.bfloat16, device=cuda), torch.empty(1, 16, device=cuda)
        plans.append((T.plan_block_attention(out, query.to(cuda), dev[0], dev[1], dev[2], dev[3], 128 ** -0.5, 1, 3000, dev[4], dev[5], lse=lse), out, lse))
        refs.append(O.attention(query, kc, vc, lens, table, 128 ** -0.5, 1, ks, vs))
    torch.cuda.synchronize()
    for _ in range(5):
        for (plan, out, lse), s in zip(plans, streams):
            with torch.cuda.stream(s):
                out.fill_(math.nan)
                plan.run()
    torch.cuda.synchronize()
    for (plan, out, lse), ref in zip(plans, refs):
        compare(out.cpu(), lse.cpu(), *ref, kc, vc, vs, table, 3000, 128)


def test_an_empty_batch_is_no_error(cuda):
    import triton_op_amd as T

    kc, vc = torch.zeros(2, 1, 8, 16, 16, device=cuda).to(FP8), torch.zeros(2, 1, 128, 16, device=cuda).to(FP8)
    q = torch.empty(0, 8, 128, dtype=torch.bfloat16, device=cuda)
    lens, table = torch.empty(0, dtype=torch.int32, device=cuda), torch.empty(0, 4, dtype=torch.int32, device=cuda)
    box = torch.zeros(2, 1, 2, 128, dtype=torch.bfloat16, device=cuda)
    T.paged_block_attention(torch.empty_like(q), q, kc, vc, lens, table, 1.0, 1, 64)
    T.key_block_bounds(box, kc, lens, table, 64)
    sel, cnt = T.select_blocks(q, box, lens, table, 3, 16, 1, 64)
    assert sel.shape == (0, 1, 3) and cnt.shape == (0, 1)


def test_max_sequence_length_beyond_the_table_is_the_tables_reach(cuda):
    """Serving code passes the model's longest context: the call is cut at what the block table holds."""
    g = torch.Generator().manual_seed(21)
    lens = torch.tensor([200, 48], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(g, 20, 2, 128, 16, "block")
    table = make_table(g, lens, 16, 20)
    query = torch.randn(2, 16, 128, generator=g).to(torch.bfloat16)
    for longest in (200, 1 << 20, 1 << 40):
        check(cuda, query, kc, vc, lens, table, 1, ks, vs, max_len=longest)
        check_select(cuda, query, _box(g, 20, 2, 128), lens, table, 4, 16, 1, max_len=longest)
    import triton_op_amd as T

    got = torch.zeros(20, 2, 2, 128, dtype=torch.bfloat16)
    want, dev = got.clone(), got.to(cuda)
    T.key_block_bounds(dev, kc.to(cuda), lens.to(cuda), table.to(cuda), 1 << 40, ks.to(cuda))
    O.bounds(want, kc, lens, table, ks)
    assert torch.equal(dev.cpu(), want)


def test_selection_without_a_query_row_takes_the_lowest_blocks(cuda):
    g = torch.Generator().manual_seed(22)
    lens = torch.tensor([16 * 30, 16 * 40], dtype=torch.int32)
    box, table = _box(g, 80, 1, 64), make_table(g, lens, 16, 80)
    query = torch.randn(2, 8, 64, generator=g).to(torch.bfloat16)
    check_select(cuda, query, box, lens, table, 9, 16, 2, 1, 3, torch.tensor([0, 2], dtype=torch.int32))
