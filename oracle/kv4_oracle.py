"""The 4-bit K/V pool and the attention over it in 64 bits on the CPU, from the definition of the format.

A pool is ``(num_blocks, num_kv_heads, 9 * head_dim / 2)`` elements of a 16-bit type: per block of sixteen slots and per head
the codes of sixteen rows, then sixteen rows of (scale, bias) pairs, one for every 64 elements.  In a group of 64:
``bias`` = min, ``scale`` = (max - min) / 15 in the 16-bit type (0 below 2^-100), ``code`` = min(15, rint((x - bias) / scale)).
Word ``r * (head_dim / 64) + g`` of a row holds elements ``64 g + 8 r + e``, e = 0 .. 7, in nibble ``e / 2 + 4 (e % 2)``.
What is held lies within +-2^15: larger numbers are stored as that, NaN as 0.
"""
from __future__ import annotations

import math

import numpy as np
import torch

ROWS, GROUP, LARGEST = 16, 64, 2.0 ** 15


def quantise(x: torch.Tensor):
    """(codes, scale, bias) of rows ``(..., head_dim)`` of a 16-bit type; scale and bias in that type, per group."""
    g = torch.nan_to_num(x.double(), nan=0.0).clamp(-LARGEST, LARGEST).unflatten(-1, (-1, GROUP))
    lo, hi = g.min(-1).values, g.max(-1).values
    scale = ((hi - lo) / 15).float().to(x.dtype)
    scale[scale.double() < 2.0 ** -100] = 0
    s = scale.double()[..., None]
    codes = torch.where(s > 0, torch.round((g - lo[..., None]) / torch.where(s > 0, s, torch.ones_like(s))), 0 * g)
    return codes.clamp(max=15).to(torch.uint8), scale, lo.to(x.dtype)


def values(codes, scale, bias) -> torch.Tensor:
    return (codes.double() * scale.double()[..., None] + bias.double()[..., None]).flatten(-2)


def _places(d: int):
    """(byte of a row, shift in it) of every element."""
    g, rest = np.divmod(np.arange(d), GROUP)
    r, e = np.divmod(rest, 8)
    nibble = e // 2 + 4 * (e % 2)
    return torch.from_numpy(4 * (r * (d // GROUP) + g) + nibble // 2), torch.from_numpy(4 * (nibble % 2))


def write(pool: torch.Tensor, rows: torch.Tensor, slots) -> None:
    """Quantise ``rows (n, heads, d)`` into ``slots`` of a CPU pool; slots outside it are dropped."""
    n, heads, d = rows.shape
    raw = pool.view(torch.uint8).view(pool.shape[0], heads, 9 * d)
    codes, scale, bias = quantise(rows)
    codes = codes.flatten(-2)
    byte, shift = _places(d)
    for i, slot in enumerate(slots):
        if not 0 <= slot < pool.shape[0] * ROWS:
            continue
        b, r = divmod(int(slot), ROWS)
        row = torch.zeros(heads, d // 2, dtype=torch.int32)
        row.index_add_(1, byte, codes[i].int() << shift.int())
        raw[b, :, r * (d // 2):(r + 1) * (d // 2)] = row.to(torch.uint8)
        pairs = torch.stack((scale[i], bias[i]), -1).flatten(1).contiguous().view(torch.uint8)
        raw[b, :, 8 * d + r * (d // 16):8 * d + (r + 1) * (d // 16)] = pairs


def read(pool: torch.Tensor, slots) -> torch.Tensor:
    """float64 values ``(n, heads, d)`` of ``slots``; zeros for those outside the pool."""
    heads, d = pool.shape[1], pool.shape[2] // 9 * 2
    raw = pool.cpu().contiguous().view(torch.uint8).view(pool.shape[0], heads, 9 * d)
    slots = torch.as_tensor(slots).long().cpu()
    ok = (slots >= 0) & (slots < pool.shape[0] * ROWS)
    s = torch.where(ok, slots, 0 * slots)
    byte, shift = _places(d)
    codes = (raw[..., :8 * d].unflatten(-1, (ROWS, d // 2))[s // ROWS, :, s % ROWS][..., byte].int() >> shift.int()) & 15
    pairs = raw[..., 8 * d:].unflatten(-1, (ROWS, d // 16))[s // ROWS, :, s % ROWS].contiguous().view(pool.dtype)
    scale, bias = pairs.unflatten(-1, (-1, 2)).double().unbind(-1)
    out = (codes.unflatten(-1, (-1, GROUP)).double() * scale[..., None] + bias[..., None]).flatten(-2)
    return torch.where(ok[:, None, None], out, 0 * out)


def attention(q, k_pool, v_pool, slots, seen, scale, device="cpu"):
    """One sequence: q ``(n, hq, d)``, its slot ids in order, ``seen (n, len(slots))``.  Returns float64 outputs and, for bounds,
    the sum of the weights times the largest of |v|, and of its group's range, and sum over d of |q k| scale, the largest over keys seen, per row and head."""
    q, seen = q.double().to(device), seen.to(device)
    n, hq, d = q.shape
    k, v = read(k_pool, slots).to(device), read(v_pool, slots).to(device)
    rep = hq // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    span = v.unflatten(-1, (-1, GROUP))
    span = ((span.max(-1).values - span.min(-1).values)[..., None]).expand_as(span.unsqueeze(-1)[..., 0]).flatten(-2)
    if k.shape[0] == 0:
        z = torch.zeros(n, hq, d, dtype=torch.float64)
        return z, z.clone(), z[..., 0].clone()
    score = torch.einsum("nhd,thd->hnt", q, k) * scale
    score = score.masked_fill(~seen[None], -math.inf)
    w = torch.softmax(score, -1).nan_to_num(0.0)                      # (rows without a key: zeros)
    size = torch.einsum("nhd,thd->hnt", q.abs(), k.abs()) * abs(scale)
    return (torch.einsum("hnt,thd->nhd", w, v).cpu(), torch.einsum("hnt,thd->nhd", w, torch.maximum(v.abs(), span)).cpu(),
            size.masked_fill(~seen[None], 0).amax(-1).T.cpu())
