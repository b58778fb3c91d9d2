"""CPU oracle of the block-granular operators, in 64 bits and in plain loops over sequences, heads and blocks: attention
over a paged cache with one scale per (block, head) (or per token, per tensor, none), the write into it, block bounds,
block selection, and attention over selected blocks.  Test infrastructure only; nothing in the package calls it."""
from __future__ import annotations

import math
from typing import Optional

import torch

FP8_MAX = 448.0
F64 = torch.float64


def key_tokens(cache: torch.Tensor) -> torch.Tensor:
    """[n, Hkv, D/x, bs, x] -> [n, Hkv, bs, D] in 64 bits"""
    return cache.to(F64).permute(0, 1, 3, 2, 4).flatten(3)


def value_tokens(cache: torch.Tensor) -> torch.Tensor:
    """[n, Hkv, D, bs] or transposed [n, Hkv, bs/x, D, x] -> [n, Hkv, bs, D] in 64 bits"""
    if cache.dim() == 5:
        return cache.to(F64).permute(0, 1, 2, 4, 3).flatten(2, 3)
    return cache.to(F64).transpose(2, 3)


def attention(query, key_cache, value_cache, lens, table, softmax_scale, q_len, key_scale=None, value_scale=None,
              selected: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None, q_lens=None, max_len=None):
    """(output [B, rows, D], lse [B, rows], logit size [B, rows]): the last is max_t sum_d |q_d k_td| * softmax_scale, what
    the rounding of a 32-bit dot product is relative to."""
    batch, rows, d = query.shape
    hkv, bs, nblk = key_cache.shape[1], key_cache.shape[3], key_cache.shape[0]
    g = rows // hkv // q_len
    k_all, v_all = key_tokens(key_cache), value_tokens(value_cache)
    if key_scale is not None:
        k_all = k_all * key_scale.to(F64)
        v_all = v_all * value_scale.to(F64)
    out = torch.zeros(batch, rows, d, dtype=F64)
    lse = torch.full((batch, rows), -math.inf, dtype=F64)
    size = torch.zeros(batch, rows, dtype=F64)
    for b in range(batch):
        n = max(0, min(int(lens[b]), table.shape[1] * bs, max_len if max_len is not None else 1 << 40))
        qb = q_len if q_lens is None else int(q_lens[b])
        blocks = -(-n // bs)
        for h in range(hkv):
            if selected is None:
                mine = list(range(blocks))
            else:
                mine = selected[b, h].tolist()[: None if counts is None else int(counts[b, h])]
                mine = [i for i in mine if 0 <= i < blocks]
            mine = [i for i in mine if 0 <= int(table[b, i]) < nblk]
            if not mine:
                continue
            at = torch.tensor(mine)
            page = table[b].long()[at]
            pos = (at[:, None] * bs + torch.arange(bs)).flatten()
            k, v = k_all[page, h].reshape(-1, d)[pos < n], v_all[page, h].reshape(-1, d)[pos < n]
            pos = pos[pos < n]
            for t in range(qb):
                seen = pos < n - (qb - 1 - t)
                if not bool(seen.any()):
                    continue
                r = h * q_len * g + t * g
                q = query[b, r:r + g].to(F64)
                logit = q @ k[seen].T * softmax_scale
                lse[b, r:r + g] = torch.logsumexp(logit, 1)
                out[b, r:r + g] = torch.softmax(logit, 1) @ v[seen]
                size[b, r:r + g] = (q.abs() @ k[seen].abs().T).amax(1) * abs(softmax_scale)
    return out, lse, size


def attention_tolerance(lse, size, tokens: int, d: int, v_max: float):
    """(bound of |output - exact| beside the final rounding, bound of |lse - exact|) of a kernel that forms logits and sums in
    32 bits and carries a probability as two bf16 terms.

    A logit is a sum of d products with exact factors (8 + 8 significant bits): at most (d + 4) 2^-24 relative to
    sum |q k| for the sum, the scales and the change to base 2; exp2 and log2 of the hardware are off by 2^-22 at most.
    A probability as hi + lo is off by (2^-8)^2 = 2^-16; sums of `tokens` terms by tokens * 2^-24 (the running rescaling by
    exp2 adds one rounding and one 2^-22 per step of 64).  Numerator and denominator each carry all of that."""
    logit = (d + 4) * 2.0**-24 * size + 2.0**-22 * (lse.abs().clamp(max=1e4) + 1)
    steps = tokens / 64 + 16
    p = logit + 2.0**-16 + tokens * 2.0**-24 + steps * 2.0**-22
    return 2 * p * v_max, logit + tokens * 2.0**-24 + steps * 2.0**-22


def block_scale(amax: float) -> float:
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    if amax == 0:
        return 2.0**-126
    return max(2.0**-126, 2.0 ** math.ceil(math.log2(amax / FP8_MAX)))


def _codes(x32: torch.Tensor) -> torch.Tensor:
    return torch.where(x32.isnan(), x32, x32.clamp(-FP8_MAX, FP8_MAX)).to(torch.float8_e4m3fn)


def write(key, value, key_cache, value_cache, slots, key_scale, value_scale):
    """The block-scaled cache write, in place on CPU tensors.  The quotient by a power of two is exact, so the only
    roundings are those to the codes; scales that are not powers of two are divided in 32 bits."""
    nblk, hkv, _, bs, _ = key_cache.shape
    d = key.shape[2]
    last = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < nblk * bs:
            last[s] = t
    by_block = {}
    for s, t in last.items():
        by_block.setdefault(s // bs, []).append((s % bs, t))
    for blk, members in by_block.items():
        off = torch.tensor([o for o, _ in members])
        tok = torch.tensor([t for _, t in members])
        for h in range(hkv):
            for x, cache, scale, is_key in ((key, key_cache, key_scale, True), (value, value_cache, value_scale, False)):
                rows = x[tok, h].float()
                fin = rows[rows.isfinite()]
                old = float(scale[blk, h, 0, 0])
                new = max(old, block_scale(float(fin.abs().max()) if fin.numel() else 0.0))
                if old > 0 and new > old:
                    ratio = torch.tensor(old, dtype=torch.float32) / torch.tensor(new, dtype=torch.float32)
                    cache[blk, h] = _codes(cache[blk, h].float() * ratio)
                code = _codes(rows / torch.tensor(new, dtype=torch.float32))
                if is_key:
                    cache[blk, h].permute(1, 0, 2)[off] = code.view(-1, d // 16, 16)
                elif cache.dim() == 5:
                    cache[blk, h].permute(0, 2, 1)[off // 16, off % 16] = code
                else:
                    cache[blk, h].transpose(0, 1)[off] = code
                scale[blk, h, 0, 0] = new


def bounds(out, key_cache, lens, table, key_scale=None, new_tokens=None, max_len=None):
    """Block bounds in place on a CPU tensor.  A key is code * scale in 32 bits (one rounding, none for a power of two)."""
    bs, nblk = key_cache.shape[3], key_cache.shape[0]
    k = key_cache.float().permute(0, 1, 3, 2, 4).flatten(3)
    if key_scale is not None:
        k = k * key_scale
    for b in range(table.shape[0]):
        n = max(0, min(int(lens[b]), table.shape[1] * bs, max_len if max_len is not None else 1 << 40))
        first = 0 if new_tokens is None else max(0, n - new_tokens) // bs
        for i in range(first, -(-n // bs)):
            page = int(table[b, i])
            if not 0 <= page < nblk:
                continue
            x = k[page][:, : min(bs, n - i * bs)]
            out[page, :, 0] = torch.where(x.isnan(), math.inf, x).amin(1).to(torch.bfloat16)
            out[page, :, 1] = torch.where(x.isnan(), -math.inf, x).amax(1).to(torch.bfloat16)


def select(query, box, lens, table, k, bs, q_len, first, recent, q_lens=None, max_len=None):
    """(selected [B, Hkv, k], counts [B, Hkv]).  Scores of bf16 numbers of ordinary range are exact in 64 bits."""
    batch, rows, d = query.shape
    hkv, nblk = box.shape[1], box.shape[0]
    g = rows // hkv // q_len
    out = torch.full((batch, hkv, k), -1, dtype=torch.int32)
    counts = torch.zeros(batch, hkv, dtype=torch.int32)
    for b in range(batch):
        n = max(0, min(int(lens[b]), table.shape[1] * bs, max_len if max_len is not None else 1 << 40))
        blocks = -(-n // bs)
        qb = q_len if q_lens is None else int(q_lens[b])
        page = table[b, :blocks].long()
        bad = (page < 0) | (page >= nblk)
        for h in range(hkv):
            q = query[b, h * q_len * g:h * q_len * g + qb * g].to(F64)
            lo, hi = box[page.clamp(0, nblk - 1), h, 0].to(F64), box[page.clamp(0, nblk - 1), h, 1].to(F64)
            s = (q.clamp(min=0)[:, None] * hi + q.clamp(max=0)[:, None] * lo).sum(2)  # [rows, blocks]
            s = torch.where(s.isnan(), -math.inf, s).clamp(max=torch.finfo(F64).max)
            s = s.amax(0) if len(q) else torch.full((blocks,), -math.inf, dtype=F64)
            s[bad] = -math.inf
            s = s.tolist()
            for i in range(blocks):
                if i < first or i >= blocks - recent:
                    s[i] = math.inf
            mine = sorted(sorted(range(blocks), key=lambda i: (-s[i], i))[:k])
            counts[b, h] = len(mine)
            out[b, h, : len(mine)] = torch.tensor(mine, dtype=torch.int32)
    return out, counts
