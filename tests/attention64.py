"""Masked attention and the 8-bit cache in 64 bits, a document at a time: what the GPU tests compare with."""

from __future__ import annotations

import math

import torch


def attend(q, k, v, *, scale=128**-0.5, causal=False, prefix=0, cap=0.0, slopes=None):
    """One document: q [n, heads, 128], k and v [m, kv heads, 128].  Returns float64 [n, heads, 128] (o, sum_j p_j |v_j|)."""
    q, k, v = q.double(), k.double(), v.double()
    n, heads, _ = q.shape
    m = k.shape[0]
    o, size = torch.zeros_like(q), torch.zeros_like(q)
    if n == 0 or m == 0:
        return o, size
    group = heads // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = scale * torch.einsum("nhd,mhd->hnm", q, k)
    if cap:
        s = cap * torch.tanh(s / cap)
    place = torch.arange(n, device=q.device)[:, None] + (m - n)
    key = torch.arange(m, device=q.device)[None]
    if slopes is not None:
        s = s - slopes.double()[:, None, None] * (place - key).abs()
    seen = (key <= place) | (key < prefix) if causal else torch.ones_like(key <= place)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(s))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)

    def mean(x):  # a weight of nothing takes nothing, not 0 x NaN
        product = torch.einsum("hnm,mhd->nhd", p, torch.nan_to_num(x, 0.0, 0.0, 0.0))
        lost = torch.einsum("hnm,mhd->nhd", (p > 0).double(), (~torch.isfinite(x)).double())
        return product.masked_fill(lost > 0, math.nan)

    return mean(v), mean(v.abs())


def attend_documents(q, k, v, bounds, key_bounds, *, prefix=None, **options):
    """Packed rows; zeros where no document has a row."""
    o, size = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    for d in range(len(bounds) - 1):
        rows, keys = slice(bounds[d], bounds[d + 1]), slice(key_bounds[d], key_bounds[d + 1])
        o[rows], size[rows] = attend(q[rows], k[keys], v[keys], prefix=prefix[d] if prefix else 0, **options)
    return o, size


def cached_rows(codes, scales, table, length):
    """float64 [length, heads, 128] of one sequence."""
    blocks = table[: -(-length // 64)].long()
    x = codes[blocks].double() * scales[blocks].double()[..., None, None]
    return x.transpose(1, 2).reshape(-1, x.shape[1], 128)[:length]


def append(codes, scales, x, table, before):
    """A sequence's new rows x [n, heads, 128] (fp32) behind ``before`` tokens, in place; the arithmetic of the definition."""
    for b in range(before // 64, -(-(before + len(x)) // 64)) if len(x) else ():
        block = int(table[b])
        low, high = max(0, 64 * b - before), min(len(x), 64 * b + 64 - before)
        kept = max(0, before - 64 * b)
        need = (x[low:high].abs().amax((0, 2)) * (1 / 127)).clamp(min=1e-10)
        scale = torch.maximum(need, scales[block]) if kept else need
        if kept:
            ratio = (scales[block] / scale)[:, None, None]
            codes[block][:, :kept] = torch.round(codes[block][:, :kept].float() * ratio).to(torch.int8)
        fresh = torch.round(x[low:high] / scale[None, :, None]).clamp(-127, 127).to(torch.int8)
        codes[block][:, kept : kept + high - low] = fresh.transpose(0, 1)
        scales[block] = scale
