"""The block-granular operators around paged decode, as cases to time and compare.

Four operators over the paged KV cache (key_cache [blocks, Hkv, D/x, bs, x], value_cache [blocks, Hkv, D, bs] or
transposed [blocks, Hkv, bs/x, D, x]; x = 16 / element size):

  write   new tokens into an FP8 cache that holds one scale per (block, kv head); a scale only grows, by powers of two,
          and the codes already in the block follow it
  attend  decode attention over such a cache (or a bf16 one), with the log-sum-exp of every row
  bounds  the smallest and largest key of every block, per kv head and head dimension
  sparse  the blocks with the largest bound of q . k are selected for each (sequence, kv head), and the attention reads
          those alone

`run` computes a case in elementary torch operations, or, where `own` is true, through the framework's entry points.
"""
import math
import random

import torch

own = False

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0


def device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 64 sequences: every sequence appends one token somewhere inside a block
        dict(name="write_step_b64", op="write", batch=64, hkv=8, d=128, bs=16, start=1000, new=1, vt=False),
        # a chunk of prompts: 4 x 2048 tokens, the first of them behind tokens that are already there
        dict(name="write_prompt_8k", op="write", batch=4, hkv=8, d=128, bs=16, start=37, new=2048, vt=False),
        # latency: a few short sequences, 8 query heads on one kv head
        dict(name="attend_b4_1k", op="attend", kv="block", batch=4, hkv=1, g=8, q=1, ragged=False, d=128, bs=16, lo=1, hi=1024, vt=False),
        # the headline batch: 64 sequences of 4096 tokens, 64 query heads on 8 kv heads
        dict(name="attend_b64_4k", op="attend", kv="block", batch=64, hkv=8, g=8, q=1, ragged=False, d=128, bs=16, lo=4096, hi=4096, vt=False),
        # a ragged batch with 1 to 4 new tokens for each sequence, 16 query heads on a kv head, large blocks
        dict(name="attend_mtp4_ragged", op="attend", kv="block", batch=32, hkv=8, g=16, q=4, ragged=True, d=128, bs=1024, lo=17, hi=8191, vt=True),
        # few long sequences
        dict(name="attend_b4_128k", op="attend", kv="block", batch=4, hkv=8, g=8, q=1, ragged=False, d=128, bs=16, lo=131072, hi=131072, vt=False),
        # after a prompt: the bounds of all blocks of 64 sequences
        dict(name="bounds_prompt_b64", op="bounds", batch=64, hkv=8, d=128, bs=16, lo=4001, hi=4096, new=0),
        # after a decode step: the bounds of the blocks that hold the two newest tokens
        dict(name="bounds_step_b64", op="bounds", batch=64, hkv=8, d=128, bs=16, lo=900, hi=4096, new=2),
        # latency: one sequence, one kv head
        dict(name="sparse_b1_2k", op="sparse", kv="block", batch=1, hkv=1, g=8, q=1, ragged=False, d=128, bs=16, lo=2047, hi=2047, vt=False, k=32, first=1, recent=2),
        # the headline batch, a quarter of its blocks
        dict(name="sparse_b64_4k", op="sparse", kv="block", batch=64, hkv=8, g=8, q=1, ragged=False, d=128, bs=16, lo=3000, hi=4096, vt=False, k=64, first=1, recent=4),
        # a 16-bit cache with two new tokens, head size 64, blocks of 64 tokens; some sequences have fewer blocks than k
        dict(name="sparse_bf16_mtp2", op="sparse", kv="bf16", batch=24, hkv=4, g=6, q=2, ragged=True, d=64, bs=64, lo=300, hi=20001, vt=False, k=24, first=1, recent=2),
        # few long sequences, 4096 tokens of 131072
        dict(name="sparse_b4_128k", op="sparse", kv="block", batch=4, hkv=8, g=8, q=1, ragged=False, d=128, bs=16, lo=131072, hi=131072, vt=False, k=256, first=4, recent=16),
    ]


def draw(rng):
    def spread(lo, hi):  # whole numbers, even over their logarithm
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["write", "attend", "attend", "bounds", "sparse", "sparse"])
    d, bs, hkv = rng.choice([64, 128, 128, 256]), rng.choice([16, 16, 64, 1024]), spread(1, 8)
    batch = spread(1, 64)
    if op == "write":
        new = spread(1, min(2048, 8192 // batch))
        return dict(op=op, batch=batch, hkv=hkv, d=d, bs=bs, start=rng.randrange(0, 2000), new=new, vt=rng.random() < 0.5)
    q, g = rng.choice([1, 1, 1, 2, 3, 4]), rng.choice([1, 2, 4, 5, 8, 8, 12, 16])
    # tokens of a sequence: no more work than the largest listed case
    hi = spread(2, min(131072, 4 * 131072 * 8 * 128 // (batch * hkv * d * max(1, q * g // 8))))
    lo = rng.choice([1, hi, rng.randrange(1, hi + 1)])
    if op == "bounds":
        return dict(op=op, batch=batch, hkv=hkv, d=d, bs=bs, lo=lo, hi=hi, new=rng.choice([0, 0, 1, 2, 4]))
    lo = max(lo, q)
    hi = max(hi, lo)
    case = dict(op=op, kv=rng.choice(["block", "block", "block", "bf16"]), batch=batch, hkv=hkv, g=g, q=q, ragged=q > 1 and rng.random() < 0.5,
                d=d, bs=bs, lo=lo, hi=hi, vt=rng.random() < 0.3)
    if op == "sparse":
        first, recent = rng.choice([0, 1, 2]), 1 + -(-(q - 1) // bs) + rng.choice([0, 1, 3])
        k = first + recent + spread(1, max(1, min(256, hi // bs)))
        case.update(k=k, first=first, recent=recent)
    return case


def lengths(case):
    """Tokens of every sequence: part of the case, the same for every seed."""
    r = random.Random("%(batch)d %(lo)d %(hi)d" % case)
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]


def new_tokens(case):
    """New tokens of every sequence (1 .. q)."""
    r = random.Random("%(batch)d %(q)d" % case)
    return [r.randint(1, case["q"]) if case["ragged"] else case["q"] for _ in range(case["batch"])]


def work(case):
    h, d, bs = case["hkv"], case["d"], case["bs"]
    if case["op"] == "write":
        tokens = case["batch"] * case["new"]
        pages = sum(1 for _ in range(case["batch"]) for p in range(case["start"] // bs, (case["start"] + case["new"] - 1) // bs + 1))
        # the rows once, their codes once, the slots, and the blocks' scales read and written
        return {"bytes": tokens * (2 * h * d * 2 + 2 * h * d + 8) + pages * h * 2 * 8, "flops": 4 * tokens * h * d}
    lens = lengths(case)
    pages = sum(-(-n // bs) for n in lens)
    if case["op"] == "bounds":
        if case["new"]:
            first = [max(0, n - case["new"]) // bs for n in lens]
            tokens = sum(n - f * bs for n, f in zip(lens, first))
            pages = sum(-(-n // bs) - f for n, f in zip(lens, first))
        else:
            tokens = sum(lens)
        # the keys, the scales and the table once, the two bounds written
        return {"bytes": tokens * h * d + pages * (h * (4 + 4 * d) + 4), "flops": 2 * tokens * h * d}
    esz = 1 if case["kv"] == "block" else 2
    rows = case["g"] * case["q"]
    io = case["batch"] * h * rows * (2 * d * 2 + 4)
    per_token = 2 * d * esz
    per_page = 8 if case["kv"] == "block" else 0
    if case["op"] == "attend":
        return {"bytes": sum(lens) * h * per_token + pages * (h * per_page + 4) + io, "flops": 4 * sum(lens) * h * rows * d}
    # every block's bounds, the selected list, and the tokens of the selected blocks
    chosen = [min(-(-n // bs), case["k"]) for n in lens]
    tokens = [min(n, c * bs) for n, c in zip(lens, chosen)]
    return {"bytes": pages * (h * 4 * d + 4) + case["batch"] * h * (case["k"] + 1) * 4 + sum(tokens) * h * per_token + sum(chosen) * h * per_page + io,
            "flops": 4 * pages * h * rows * d + 4 * sum(tokens) * h * rows * d}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def generator(seed, tag):
    return torch.Generator(device=device()).manual_seed(seed * 1000 + tag)


def power_of_two_scale(amax):
    """The smallest power of two s with amax <= 448 s (at least 2^-126)."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.full_like(amax, 2.0**-126))


def key_layout(x):
    """[n, Hkv, bs, D] -> [n, Hkv, D/x, bs, x]"""
    n, h, bs, d = x.shape
    e = 16 // x.element_size()
    return x.view(n, h, bs, d // e, e).permute(0, 1, 3, 2, 4)


def value_layout(x, vt):
    """[n, Hkv, bs, D] -> [n, Hkv, D, bs], or transposed [n, Hkv, bs/x, D, x]"""
    n, h, bs, d = x.shape
    e = 16 // x.element_size()
    return x.view(n, h, bs // e, e, d).permute(0, 1, 2, 4, 3) if vt else x.transpose(2, 3)


def key_tokens(x):
    """[..., D/x, bs, x] -> [..., bs, D]"""
    return x.transpose(-3, -2).flatten(-2)


def value_tokens(x, vt):
    """[..., D, bs], or transposed [..., bs/x, D, x] -> [..., bs, D]"""
    return x.transpose(-2, -1).flatten(-3, -2) if vt else x.transpose(-2, -1)


def prepare(case, seed):
    dev = device()
    h, d, bs, batch = case["hkv"], case["d"], case["bs"], case["batch"]
    write = case["op"] == "write"
    lens = [case["start"] + case["new"]] * batch if write else lengths(case)
    need = [-(-n // bs) for n in lens]
    blocks = int(sum(need) * 1.25) + 1
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.empty(batch, max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):  # a row's unused entries name its first block
        table[b, :n] = order[at:at + n]
        table[b, n:] = order[at]
        at += n
    table = table.to(dev)
    # keys and values: N(0, 1) with a magnitude for each (block, head), as the channels and layers of a model differ
    kv = case.get("kv", "block")
    vt = case.get("vt", False)
    dtype = FP8 if kv == "block" else torch.bfloat16
    e = 16 if kv == "block" else 8
    kc = torch.empty(blocks, h, d // e, bs, e, dtype=dtype, device=dev)
    vc = torch.empty((blocks, h, bs // e, d, e) if vt else (blocks, h, d, bs), dtype=dtype, device=dev)
    ks, vs = (torch.empty(blocks, h, 1, 1, device=dev) for _ in range(2)) if kv == "block" else (None, None)
    bounds = torch.zeros(blocks, h, 2, d, dtype=torch.bfloat16, device=dev)
    step = max(1, (1 << 27) // (h * bs * d))
    gen = generator(seed, 1)
    for lo in range(0, blocks, step):
        n = min(step, blocks - lo)
        for cache, scale, lay in ((kc, ks, key_layout), (vc, vs, lambda x: value_layout(x, vt))):
            x = torch.randn(n, h, bs, d, generator=gen, device=dev)
            x *= torch.randn(n, h, 1, 1, generator=gen, device=dev).mul_(0.4).exp_()
            if kv == "block":
                s = power_of_two_scale(x.abs().amax((2, 3), keepdim=True))
                c = (x / s).clamp_(-FP8_MAX, FP8_MAX).to(FP8)
                cache[lo:lo + n] = lay(c)
                scale[lo:lo + n] = s
                x = c.float() * s
            else:
                x = x.to(dtype)
                cache[lo:lo + n] = lay(x)
            if cache is kc and case["op"] != "write" and not (case["op"] == "bounds" and case["new"] == 0):
                bounds[lo:lo + n] = torch.stack((x.amin(2), x.amax(2)), 2).to(torch.bfloat16)
    state = dict(case=case, key_cache=kc, value_cache=vc, key_scale=ks, value_scale=vs, table=table)
    if write:
        pos = case["start"] + torch.arange(case["new"], device=dev)
        state["slots"] = (table[:, pos // bs].long() * bs + pos % bs).reshape(-1)
        for name in ("key", "value"):
            x = torch.randn(batch * case["new"], h, d, generator=gen, device=dev)
            state[name] = (x * torch.randn(batch * case["new"], h, 1, generator=gen, device=dev).mul_(0.5).exp_()).to(torch.bfloat16)
        return state
    state.update(lens=torch.tensor(lens, dtype=torch.int32, device=dev), longest=max(lens), bounds=bounds)
    if case["op"] == "bounds":
        return state
    rows = h * case["q"] * case["g"]
    state["query"] = torch.randn(batch, rows, d, generator=gen, device=dev).to(torch.bfloat16)
    state["output"] = torch.empty(batch, rows, d, dtype=torch.bfloat16, device=dev)
    state["lse"] = torch.empty(batch, rows, device=dev)
    state["q_lens"] = torch.tensor(new_tokens(case), dtype=torch.int32, device=dev) if case["ragged"] else None
    return state


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def plain_write(s):
    bs, vt = s["case"]["bs"], s["case"]["vt"]
    slots = s["slots"]
    block, off = slots // bs, slots % bs
    touched = block.unique()
    token = torch.arange(slots.numel(), device=slots.device)
    owner = torch.full((s["key_cache"].shape[0] * bs,), -1, dtype=torch.int64, device=slots.device).scatter_reduce(0, slots, token, "amax")
    kept = owner[slots] == token  # of two tokens for one slot the later one stays

    def one(x, cache, scale, key):
        x, b, o = x[kept].float(), block[kept], off[kept]
        amax = torch.zeros(scale.shape[:2], device=x.device).scatter_reduce(0, b[:, None].expand(-1, x.shape[1]), x.abs().amax(2), "amax")
        old = scale[:, :, 0, 0]
        grown = torch.maximum(old, power_of_two_scale(amax))
        new = torch.where(torch.zeros_like(old).index_fill(0, touched, 1.0) > 0, grown, old)
        ratio = torch.where(old > 0, old / new, torch.ones_like(old))
        # the codes of the touched blocks follow their scale
        cache[touched] = (cache[touched].float() * ratio[touched].view(-1, ratio.shape[1], *([1] * (cache.dim() - 2)))).to(FP8)
        code = (x / new[b].unsqueeze(2)).clamp(-FP8_MAX, FP8_MAX).to(FP8)  # [tokens, Hkv, D]
        if key:
            cache.permute(0, 3, 1, 2, 4)[b, o] = code.view(*code.shape[:2], -1, 16)
        elif vt:
            cache.permute(0, 2, 4, 1, 3)[b, o // 16, o % 16] = code
        else:
            cache.permute(0, 3, 1, 2)[b, o] = code
        scale.copy_(new.view_as(scale))

    one(s["key"], s["key_cache"], s["key_scale"], True)
    one(s["value"], s["value_cache"], s["value_scale"], False)
    return {k: s[k] for k in ("key_cache", "value_cache", "key_scale", "value_scale")}


def plain_bounds(s):
    case, lens, table = s["case"], s["lens"].long(), s["table"].long()
    bs, h, d = case["bs"], case["hkv"], case["d"]
    blocks = (lens + bs - 1) // bs
    if case["new"]:
        first = (lens - case["new"]).clamp(min=0) // bs
        at = first[:, None] + torch.arange((case["new"] + bs - 2) // bs + 1, device=lens.device)
    else:
        at = torch.arange(table.shape[1], device=lens.device).expand(len(lens), -1)
    live = at < blocks[:, None]
    at, seq = at[live], torch.arange(len(lens), device=lens.device)[:, None].expand_as(live)[live]
    page = table[seq, at]
    x = key_tokens(s["key_cache"][page].float()) * s["key_scale"][page]  # [n, Hkv, bs, D]
    gone = (at[:, None] * bs + torch.arange(bs, device=lens.device) >= lens[seq][:, None])[:, None, :, None] | x.isnan()
    lo = x.masked_fill(gone, math.inf).amin(2)
    hi = x.masked_fill(gone, -math.inf).amax(2)
    s["bounds"][page] = torch.stack((lo, hi), 2).to(torch.bfloat16)
    return s["bounds"]


def plain_select(s):
    case, lens, table = s["case"], s["lens"].long(), s["table"].long()
    bs, h, k = case["bs"], case["hkv"], case["k"]
    q = s["query"].double().view(len(lens), h, -1, case["d"])
    box = s["bounds"][table].double()  # [B, P, Hkv, 2, D]
    lo, hi = box[..., 0, :].permute(0, 2, 3, 1), box[..., 1, :].permute(0, 2, 3, 1)
    score = q.clamp(min=0) @ hi + q.clamp(max=0) @ lo  # [B, Hkv, rows, P]
    row = torch.arange(q.shape[2], device=lens.device) // case["g"]
    q_lens = s["q_lens"] if s["q_lens"] is not None else torch.full_like(lens, case["q"])
    score = score.nan_to_num(nan=-math.inf, posinf=torch.finfo(torch.float64).max, neginf=-math.inf)
    score = score.masked_fill((row >= q_lens[:, None])[:, None, :, None], -math.inf).amax(2)
    blocks = ((lens + bs - 1) // bs)[:, None, None]
    at = torch.arange(table.shape[1], device=lens.device)
    score = score.masked_fill((at < case["first"]) | (at >= blocks - case["recent"]), math.inf).masked_fill(at >= blocks, -math.inf)
    chosen = score.sort(dim=-1, descending=True, stable=True).indices[..., :k]
    chosen = torch.nn.functional.pad(chosen, (0, k - chosen.shape[-1]), value=table.shape[1])
    chosen = chosen.masked_fill(chosen >= blocks, table.shape[1]).sort(dim=-1).values
    chosen = chosen.masked_fill(chosen >= table.shape[1], -1).to(torch.int32)
    return chosen, (chosen >= 0).sum(-1).to(torch.int32)


def plain_attention(s, chosen=None):
    case, lens, table = s["case"], s["lens"].long(), s["table"].long()
    bs, h, d = case["bs"], case["hkv"], case["d"]
    batch = len(lens)
    if chosen is None:
        page = table[:, None, :].expand(-1, h, -1)
        at = torch.arange(table.shape[1], device=lens.device).view(1, 1, -1)
    else:
        at = chosen.long()
        page = table[:, None, :].expand(-1, h, -1).gather(2, at.clamp(min=0))
    head = torch.arange(h, device=lens.device)[None, :, None]
    k, v = key_tokens(s["key_cache"][page, head].float()), value_tokens(s["value_cache"][page, head].float(), case["vt"])
    if s["key_scale"] is not None:
        k, v = k * s["key_scale"][page, head], v * s["value_scale"][page, head]
    k, v = k.reshape(batch, h, -1, d), v.reshape(batch, h, -1, d)
    pos = (at[..., None] * bs + torch.arange(bs, device=lens.device)).masked_fill(at[..., None] < 0, 1 << 40).flatten(2)  # [B or 1, Hkv or 1, T]
    v = v.masked_fill((pos >= lens[:, None, None])[..., None], 0.0)
    q = s["query"].float().view(batch, h, -1, d)
    logit = (q @ k.transpose(2, 3)) * d ** -0.5
    row = torch.arange(q.shape[2], device=lens.device) // case["g"]
    q_lens = s["q_lens"].long() if s["q_lens"] is not None else torch.full_like(lens, case["q"])
    end = torch.where(row < q_lens[:, None], lens[:, None] - (q_lens[:, None] - 1 - row), torch.zeros_like(row))  # [B, rows]
    logit = logit.masked_fill(pos[:, :, None, :] >= end[:, None, :, None], -math.inf)
    top = logit.amax(-1, keepdim=True)
    p = (logit - top.masked_fill(top == -math.inf, 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / total.masked_fill(total == 0, 1.0)
    return out.to(torch.bfloat16).view(batch, -1, d), (top + total.log()).view(batch, -1)


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        if op == "write":
            return plain_write(s)
        if op == "bounds":
            return plain_bounds(s)
        if op == "attend":
            return plain_attention(s)
        chosen, count = plain_select(s)
        return (chosen, count) + plain_attention(s, chosen)
    import triton_op_amd as T

    if op == "write":
        T.kv_cache_write(s["key"], s["value"], s["key_cache"], s["value_cache"], s["slots"], s["key_scale"], s["value_scale"])
        return {k: s[k] for k in ("key_cache", "value_cache", "key_scale", "value_scale")}
    if op == "bounds":
        T.key_block_bounds(s["bounds"], s["key_cache"], s["lens"], s["table"], s["longest"], s["key_scale"], new_tokens=case["new"] or None)
        return s["bounds"]
    chosen = count = None
    if op == "sparse":
        chosen, count = T.select_blocks(s["query"], s["bounds"], s["lens"], s["table"], case["k"], case["bs"], case["q"], s["longest"],
                                        first_blocks=case["first"], recent_blocks=case["recent"], query_lens=s["q_lens"])
    T.paged_block_attention(s["output"], s["query"], s["key_cache"], s["value_cache"], s["lens"], s["table"], case["d"] ** -0.5, case["q"],
                            s["longest"], s["key_scale"], s["value_scale"], selected_blocks=chosen, selected_counts=count,
                            query_lens=s["q_lens"], lse=s["lse"])
    return (s["output"], s["lse"]) if op == "attend" else (chosen, count, s["output"], s["lse"])


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f64, dev = torch.float64, s["key_cache"].device
    h, d, bs = case["hkv"], case["d"], case["bs"]

    def e4m3(x):  # the nearest value of the format, ties to the even mantissa
        a = x.abs().clamp(max=FP8_MAX)
        unit = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0**-6))) - 3)
        return torch.copysign(torch.round(a / unit) * unit, x)

    if case["op"] == "write":
        kd = s["key_cache"].to(f64).permute(0, 1, 3, 2, 4).reshape(-1, h, bs, d)
        v = s["value_cache"].to(f64)
        vd = (v.permute(0, 1, 2, 4, 3) if case["vt"] else v.transpose(2, 3)).reshape(-1, h, bs, d)
        out = {}
        for name, cache, rows in (("key", kd, s["key"]), ("value", vd, s["value"])):
            scale = s[name + "_scale"].to(f64)[:, :, 0, 0].clone()
            x = rows.to(f64)
            for blk in torch.unique(s["slots"] // bs).tolist():
                mine = torch.nonzero(s["slots"] // bs == blk)[:, 0]
                amax = x[mine].abs().amax((0, 2))
                want = torch.exp2(torch.ceil(torch.log2(amax / FP8_MAX)))
                new = torch.maximum(scale[blk], want)
                grew = new > scale[blk]
                cache[blk][grew] = e4m3(cache[blk][grew] * (scale[blk] / new)[grew][:, None, None])
                cache[blk][:, (s["slots"][mine] % bs)] = e4m3(x[mine] / new[None, :, None]).transpose(0, 1)
                scale[blk] = new
            out[name + "_scale"] = scale.view(-1, h, 1, 1)
        out["key_cache"] = kd.view(-1, h, bs, d // 16, 16).permute(0, 1, 3, 2, 4).contiguous()
        out["value_cache"] = (vd.view(-1, h, bs // 16, 16, d).permute(0, 1, 2, 4, 3) if case["vt"] else vd.transpose(2, 3)).contiguous()
        return out

    lens, table = s["lens"].tolist(), s["table"].long()
    if case["op"] == "bounds":
        out = s["bounds"].to(f64)
        for b, n in enumerate(lens):
            lo = max(0, n - case["new"]) // bs if case["new"] else 0
            page = table[b, lo:-(-n // bs)]
            x = s["key_cache"][page].to(f64).permute(0, 3, 1, 2, 4).reshape(-1, h, d) * s["key_scale"][page].to(f64).expand(-1, h, bs, 1).transpose(1, 2).reshape(-1, h, 1)
            for i in (range(len(page)) if case["new"] else ()):
                y = x[i * bs:min((i + 1) * bs, n - lo * bs)]
                out[page[i], :, 0], out[page[i], :, 1] = y.amin(0), y.amax(0)
            if not case["new"]:
                full, rest = n // bs, n % bs
                y = x[:full * bs].view(full, bs, h, d)
                if full:
                    out[page[:full], :, 0], out[page[:full], :, 1] = y.amin(1), y.amax(1)
                if rest:
                    out[page[full], :, 0], out[page[full], :, 1] = x[full * bs:n].amin(0), x[full * bs:n].amax(0)
        return out

    q_lens, g, q = new_tokens(case), case["g"], case["q"]
    out = torch.zeros(len(lens), h, q * g, d, dtype=f64, device=dev)
    lse = torch.full((len(lens), h, q * g), -math.inf, dtype=f64, device=dev)
    picked = torch.full((len(lens), h, case.get("k", 0)), -1, dtype=torch.int32, device=dev)
    for b, n in enumerate(lens):
        rows = s["query"][b].to(f64).view(h, q * g, d)[:, :q_lens[b] * g]
        pages = -(-n // bs)
        if case["op"] == "sparse":
            box = s["bounds"][table[b, :pages]].to(f64)  # [P, Hkv, 2, D]
            every = rows.clamp(min=0) @ box[:, :, 1].permute(1, 2, 0) + rows.clamp(max=0) @ box[:, :, 0].permute(1, 2, 0)
            every = every.amax(1)
            every[:, :case["first"]] = math.inf
            every[:, max(0, pages - case["recent"]):] = math.inf
        for head in range(h):
            if case["op"] == "sparse":
                rank = every[head].tolist()
                mine = sorted(sorted(range(pages), key=lambda i: (-rank[i], i))[:case["k"]])
                picked[b, head, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
                mine = torch.tensor(mine, device=dev)
            else:
                mine = torch.arange(pages, device=dev)
            page = table[b, mine]
            k = s["key_cache"][page, head].to(f64).transpose(1, 2).reshape(-1, bs, d)
            v = s["value_cache"][page, head].to(f64)
            v = (v.transpose(2, 3) if case["vt"] else v.transpose(1, 2)).reshape(-1, bs, d)
            if s["key_scale"] is not None:
                k, v = k * s["key_scale"][page, head].to(f64), v * s["value_scale"][page, head].to(f64)
            pos = (mine[:, None] * bs + torch.arange(bs, device=dev)).flatten()
            k, v, pos = k.reshape(-1, d)[pos < n], v.reshape(-1, d)[pos < n], pos[pos < n]
            logit = rows[head] @ k.T / math.sqrt(d)
            end = n - (q_lens[b] - 1 - torch.arange(q_lens[b] * g, device=dev) // g)
            logit[pos[None, :] >= end[:, None]] = -math.inf
            lse[b, head, :q_lens[b] * g] = torch.logsumexp(logit, 1)
            out[b, head, :q_lens[b] * g] = torch.softmax(logit, 1) @ v
    out, lse = out.view(len(lens), -1, d), lse.view(len(lens), -1)
    if case["op"] == "attend":
        return out, lse
    return picked, (picked >= 0).sum(-1).to(torch.int32), out, lse
