"""The 8-bit paged cache's operators from their definitions, in 64 bits on the CPU, with error bounds.

Written a page and a row at a time, for small sizes. Values of the cache are held as float64 beside the
codes, so attention starts from exactly what the cache stands for.
"""
import math

import torch

E4M3 = torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a step, relative


def power_for(amax: float) -> float:
    """The smallest 2^e, e >= -126, with amax <= 448 * 2^e; 0 for 0."""
    if amax == 0:
        return 0.0
    e = -126
    while amax > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def nearest_code(x, scale):
    """e4m3 codes (uint8) of float64 x at ``scale``: nearest, ties to even; finite beyond 448 and infinities: 448.

    At scale 0 (no finite value but zeros) any code stands for 0; it is the one at scale 1.
    """
    ratio = x / (scale or 1.0)
    table = torch.arange(0x7F, dtype=torch.uint8).view(E4M3).to(torch.float64)      # every finite size in order
    size = ratio.abs().clamp(max=448.0).nan_to_num(nan=0.0)
    high = torch.searchsorted(table, size.contiguous()).clamp(max=0x7E)
    low = (high - 1).clamp(min=0)
    up, down = table[high] - size, size - table[low]
    code = torch.where((up < down) | ((up == down) & (high % 2 == 0)), high, low)
    code = torch.where(x.isnan(), torch.full_like(code, 0x7F), code)
    return torch.where(x.isnan(), code, code + 128 * torch.signbit(ratio).to(code.dtype)).to(torch.uint8)


def rotate(x, positions, rotary_dim, base, interleaved):
    """x float64 [rows, heads, dim] turned by the angles of its positions."""
    out = x.clone()
    half = rotary_dim // 2
    for r, p in enumerate(positions):
        for i in range(half):
            angle = p * float(base) ** (-2 * i / rotary_dim)
            # the table's float32 cosine and sine are the operator's inputs
            c = torch.tensor(math.cos(angle), dtype=torch.float32).item()
            s = torch.tensor(math.sin(angle), dtype=torch.float32).item()
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            out[r, :, a] = x[r, :, a] * c - x[r, :, b] * s
            out[r, :, b] = x[r, :, b] * c + x[r, :, a] * s
    return out


def rows_of(start, lengths):
    """(sequence, row, position) of every row that is a sequence's."""
    for s in range(len(lengths)):
        for row in range(start[s], start[s + 1]):
            yield s, row, lengths[s] - (start[s + 1] - row)


def attend(query, codes, scales, table, start, lengths, block_size, scale):
    """(out, bound) float64 [rows, q_heads, dim]; rows without a token are 0, others' bound also counts the rounding.

    The bound of one output: weights reach 16 bits once (half a step of fp16, 2^-11, and an absolute 2^-25
    where they are below fp16's normal numbers; the largest unnormalised weight is at least 1); scores are
    32-bit sums of head_dim products, exponentials and sums 32-bit; the result is rounded once to its type.
    """
    rows, q_heads, dim = query.shape
    group = q_heads // codes.shape[3]
    q = query.to(torch.float64)
    out = torch.zeros(rows, q_heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    cached = {}
    for s, row, position in rows_of(start, lengths):
        if position < 0:
            continue
        if s not in cached:
            pages = torch.tensor(table[s][: -(-lengths[s] // block_size)])
            held = codes.view(E4M3)[:, pages].to(torch.float64)
            held = held * scales[pages].to(torch.float64).permute(1, 0, 2)[:, :, None, :, None]
            cached[s] = held.flatten(1, 2)
        kv = cached[s][:, : position + 1].repeat_interleave(group, dim=2)          # [2, tokens, q_heads, dim]
        score = torch.einsum("hd,thd->ht", q[row], kv[0]) * scale
        size = torch.einsum("hd,thd->ht", q[row].abs(), kv[0].abs()).amax(dim=1) * scale
        weight = torch.softmax(score, dim=-1)
        out[row] = torch.einsum("ht,thd->hd", weight, kv[1])
        spread = torch.einsum("ht,thd->hd", weight, kv[1].abs())
        # score error: dim + 4 roundings of 2^-24 of the products' size, twice (numerator and sum)
        relative = 2.0 ** -11 + 2 * (dim + 4) * 2.0 ** -24 * size + (position + 65) * 2.0 ** -24 + 2.0 ** -20
        total = torch.exp(score - score.amax(dim=-1, keepdim=True)).sum(dim=-1)
        faint = 2.0 ** -25 * kv[1].abs().sum(dim=0) / total[:, None]
        bound[row] = relative[:, None] * spread + faint
    half = HALF[query.dtype]
    tiny = 2.0 ** -25 if query.dtype == torch.float16 else 0.0                  # below fp16's normal numbers
    return out, bound * (1 + half) + half * out.abs() + tiny
