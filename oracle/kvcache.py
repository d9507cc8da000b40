"""CPU oracle of the 4-bit paged cache and of cache eviction, in 64 bits.

Test infrastructure, like oracle/reference.py: plain restatements of the
operators' definitions (include/attn_b200.h), one sequence and one head at a time.
"""
from __future__ import annotations

import math

import numpy as np
import torch

GROUP = 32


def row_bytes(d):
    return d // 2 + d // 8


def code_places(d, value):
    """(byte, shift) of the code of every dim in a K row, or in a V row (value=True)."""
    ng = d // GROUP
    byte, shift = np.zeros(d, dtype=np.int64), np.zeros(d, dtype=np.int64)
    for i in range(d):
        w, r = divmod(i, GROUP)
        if value:
            bit = 16 * ((r // 4) * ng + w) + 4 * (r % 4)
        else:
            bit = 32 * ((r // 8) * ng + w) + 4 * (r % 8)
        byte[i], shift[i] = bit // 8, bit % 8
    return byte, shift


def quantise(x):
    """x [..., D] fp16 or bf16 -> (codes int64 [..., D], scales fp16, lows fp16 [..., NG])."""
    g = x.cpu().double().unflatten(-1, (-1, GROUP))
    bad = ~(g.abs() <= 65504).all(-1)
    low = g.amin(-1).to(torch.float16)
    scale = ((g.amax(-1) - low.double()).float() / 15).to(torch.float16)
    step = scale.double()[..., None]
    code = torch.where(step > 0, ((g - low.double()[..., None]) / step).nan_to_num(0).round(),
                       torch.zeros_like(g)).clamp(0, 15)
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    nan = torch.full_like(low, math.nan)
    return code.long().flatten(-2), torch.where(bad, nan, scale), torch.where(bad, nan, low)


def pack(x, value):
    """Rows uint8 [..., row_bytes(D)] of x [..., D]."""
    code, scale, low = quantise(x)
    d = code.shape[-1]
    byte, shift = code_places(d, value)
    rows = np.zeros(code.shape[:-1] + (d // 2,), dtype=np.uint8)
    c = code.numpy().astype(np.uint8)
    for i in range(d):
        rows[..., byte[i]] |= c[..., i] << np.uint8(shift[i])
    par = torch.cat([scale, low], -1).contiguous().view(torch.uint8)
    return torch.cat([torch.from_numpy(rows), par], -1)


def parts(rows, value):
    """(codes, scales, lows) as fp64 [..., D] of packed rows."""
    rows = rows.cpu()
    d = rows.shape[-1] * 8 // 5
    byte, shift = code_places(d, value)
    code = (rows[..., torch.from_numpy(byte)].long() >> torch.from_numpy(shift)) & 15
    par = rows[..., d // 2:].contiguous().view(torch.float16).double()
    ng = d // GROUP
    return (code.double(), par[..., :ng].repeat_interleave(GROUP, -1),
            par[..., ng:].repeat_interleave(GROUP, -1))


def unpack(rows, value):
    code, scale, low = parts(rows, value)
    return low + scale * code


def rows_of(cache, table, n, head):
    """The first n tokens' rows of one head: cache [num_blocks, H_kv, bs, ...]."""
    bs = cache.shape[2]
    i = torch.arange(n)
    return cache[table.long()[i // bs], head, i % bs]


def slots_of(table, n, bs):
    i = torch.arange(n)
    return table.long()[i // bs] * bs + i % bs


def attend(q, k, v, scale=None):
    """q [G, D], k and v [n, D] -> (out [G, D], p [G, n]) in fp64."""
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    if k.shape[0] == 0:
        return torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[0], 0).double()
    s = q.double() @ k.double().T * scale
    p = torch.softmax(s, -1)
    return p @ v.double(), p


def select(totals, keep, recent, sinks):
    """Indices (ascending) that stay of one head's totals [n]."""
    n = len(totals)
    if n <= keep:
        return list(range(n))
    held = list(range(sinks)) + list(range(n - recent, n))
    rest = range(sinks, n - recent)
    value = [-math.inf if math.isnan(x) else x for x in map(float, totals)]
    best = sorted(rest, key=lambda i: (-value[i], i))[:keep - sinks - recent]
    return sorted(held + best)
