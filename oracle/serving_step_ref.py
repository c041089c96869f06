"""Plain 64-bit restatement of the serving-step operators, used by the tests only (CPU tensors, loops over sequences).

Written from the definitions: pages as Python lists, norm and rotation in float64, e2m1 rounding by distance to the eight magnitudes,
attention as a softmax over the visible tokens of each row.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


# ---------------------------------------------------------------------------------------------------------------- pages
def ref_alloc(cached, news, table, free, page_size, total_q):
    """``cached``, ``news``: tokens per sequence; ``table``: list of rows; ``free``: list (a stack).  Returns slots, positions, lengths,
    refused, the pages left and the new table."""
    table = [list(r) for r in table]
    slots, positions, lengths, refused = [], [], [], []
    wanted = 0  # pages asked for by the sequences that fit their rows and lie in the step, so far
    for b, (c, n) in enumerate(zip(cached, news)):
        fits = n > 0 and c >= 0 and c + n <= min(len(table[b]) * page_size, 2 ** 31 - 1) and len(slots) + n <= total_q
        need = -(-(c + n) // page_size) - -(-c // page_size) if fits else 0
        served = fits and (need == 0 or wanted + need <= len(free))
        if served:
            first = -(-c // page_size)
            for i in range(need):
                table[b][first + i] = free[len(free) - 1 - (wanted + i)]
        wanted += need
        for i in range(max(n, 0)):
            pos = c + i
            slots.append(table[b][pos // page_size] * page_size + pos % page_size if served else -1)
            positions.append(pos if served else -1)
        lengths.append(c + n if served else c)
        refused.append(n > 0 and not served)
    taken, total = 0, 0
    for b, (c, n) in enumerate(zip(cached, news)):
        if lengths[b] != c:
            taken += -(-lengths[b] // page_size) - -(-c // page_size)
    pad = total_q - len(slots)
    return (slots + [-1] * pad)[:total_q], (positions + [-1] * pad)[:total_q], lengths, refused, len(free) - taken, table


def ref_release(finished, lengths, table, free, page_size):
    free = list(free)
    out = []
    for f, n, row in zip(finished, lengths, table):
        if f:
            free += row[: -(-max(n, 0) // page_size)]
        out.append(0 if f else n)
    return out, free


# --------------------------------------------------------------------------------------------------------------- 4 bits
def ref_fp4_quantize(x: torch.Tensor):
    """``x [..., dim]`` (values of 32 bits) -> codes ``[..., dim / 2]``, scale bytes ``[..., dim / 32]``, values in float64."""
    x = x.double()
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    finite = torch.isfinite(blocks).all(-1)
    blocks = torch.where(finite[..., None], blocks, torch.zeros_like(blocks)).clamp(-3 * 2.0 ** 126, 3 * 2.0 ** 126)
    amax = blocks.abs().amax(-1)
    e = torch.full_like(amax, -126.0)
    while bool((amax > 6 * torch.exp2(e)).any()):
        e = torch.where(amax > 6 * torch.exp2(e), e + 1, e)
    size = blocks.abs() / torch.exp2(e)[..., None]
    index = torch.zeros(size.shape, dtype=torch.int64)
    for i in range(1, 8):
        mid = (E2M1[i - 1] + E2M1[i]) / 2
        index = torch.where((size > mid) | ((size == mid) & (i % 2 == 0)), i, index)
    negative = torch.signbit(blocks)
    value = torch.where(negative, -E2M1[index], E2M1[index]) * torch.exp2(e)[..., None]
    value = torch.where(finite[..., None], value, torch.full_like(value, math.nan)).reshape(x.shape)
    code = (index + 8 * negative.long()).reshape(*x.shape[:-1], -1, 2)
    byte = torch.where(finite, e + 127, torch.full_like(e, 255.0))
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), byte.to(torch.uint8), value


def ref_fp4_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    grid = torch.cat([E2M1, -E2M1])
    c = codes.long()
    x = torch.stack([grid[c % 16], grid[c // 16]], -1).reshape(*codes.shape[:-1], -1, 32)
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (x * s[..., None]).reshape(*codes.shape[:-1], -1)


# --------------------------------------------------------------------------------------------------------------- append
def ref_norm_rope(x, weight: Optional[torch.Tensor], cos, sin, positions, eps: float, interleaved: bool) -> torch.Tensor:
    """``x [tokens, heads, dim]`` -> float64."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    if cos is None:
        return y
    half = cos.shape[1]
    at = positions.long().clamp(0, cos.shape[0] - 1)
    out = y.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos[at, i].double()[:, None], sin[at, i].double()[:, None]
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
    return out


def ref_fp8_quantize(x: torch.Tensor):
    """``x [..., dim]`` (values of 32 bits) -> (e4m3fn codes, fp32 scales): scale = max(absmax, 1e-4) / 448."""
    x = x.float()
    scale = x.abs().amax(-1).clamp(min=1e-4) / torch.tensor(448.0)
    return (x / scale[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


# ------------------------------------------------------------------------------------------------------------ attention
def ref_attention(q, k, v, lens, table, page_size, *, sm_scale, softcap=0.0, causal=True):
    """``q [B, S_q, H, D]``; ``k, v [pages, H_kv, page_size, D]`` float64.  Returns (output, sum of p |v|, largest sum over a visible
    token's |k|) in float64, the last two for error bounds."""
    B, S, H, D = q.shape
    hk = k.shape[1]
    out, spread, reach = torch.zeros(B, S, H, D, dtype=torch.float64), torch.zeros(B, S, H, D, dtype=torch.float64), torch.zeros(B, S, H, 1, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        pages = table[b, : -(-n // page_size)].long()
        for h in range(H):
            kk, vv = (x[pages, h // (H // hk)].reshape(-1, D)[:n] for x in (k, v))
            for s in range(S):
                seen = min(n, n - S + s + 1) if causal else n
                if seen <= 0:
                    continue
                z = kk[:seen] @ q[b, s, h].double() * sm_scale
                if softcap:
                    z = softcap * torch.tanh(z / softcap)
                p = torch.softmax(z, 0)
                out[b, s, h] = p @ vv[:seen]
                spread[b, s, h] = p @ vv[:seen].abs()
                reach[b, s, h] = kk[:seen].abs().sum(-1).amax()
    return out, spread, reach
