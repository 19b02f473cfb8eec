"""Seeded inputs and 64-bit plain forms of the attention-side operators (`gemv`, `qk_norm_rope`, the
paged cache, `paged_attention`), shared by their tests.  Everything here is torch on whatever device its
inputs live, in float64, written from the definitions."""

from __future__ import annotations

import math

import torch

HALF = 2.0 ** -8      # largest relative error of a rounding to BF16 (eight significant bits)
SINGLE = 2.0 ** -22   # of one FP32 addition in a product (twice the unit roundoff: it may truncate)


def gemv(x, codes, scale, experts=None, top_k=1):
    """float64 [rows, N] and the sums of the terms' magnitudes.  ``experts``: a local index per row,
    negative for none."""
    x = x.double()
    rows = x.shape[0] * top_k
    out, size = [], []
    for r in range(rows):
        e = 0 if experts is None else int(experts[r])
        w = (codes[max(e, 0)].double() - 8) * scale[max(e, 0)].double().repeat_interleave(32, dim=1)
        keep = 1.0 if e >= 0 else 0.0
        out.append(keep * (w @ x[r // top_k]))
        size.append(keep * (w.abs() @ x[r // top_k].abs()))
    return torch.stack(out), torch.stack(size)


def norm_rope(x, weight, cos_sin, positions, eps, interleaved):
    x = x.double()
    y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    half = cos_sin.shape[1] // 2
    table = cos_sin.double()[positions.long()]
    out = y.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = table[:, i, None], table[:, half + i, None]
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
    return out


def angles(positions, rotary, device):
    rate = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / max(rotary, 1))
    at = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * rate
    return torch.cat([at.cos(), at.sin()], dim=1).float()


def stored(cache):
    """float64 keys and values [pages, heads, page_size, dim] that a cache stands for."""
    if cache.k_scale is None:
        return cache.k.double(), cache.v.double()
    return tuple((c.double() - 128) * s.double()[..., None] for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))


def fill(cache, g):
    """Normal values into a cache, a scale of its own for each row."""
    for pages, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        if scales is None:
            pages.copy_(torch.randn(pages.shape, generator=g, device=pages.device))
        else:
            pages.copy_(torch.randint(1, 256, pages.shape, generator=g, device=pages.device, dtype=torch.int32))
            scales.copy_(torch.rand(scales.shape, generator=g, device=pages.device) * 0.02 + 0.001)


def attention(q, k_all, v_all, tables, lengths, page_size, *, scale=None, window=None):
    """float64 (out, lse, sizes of the values' terms, sizes of the scores' terms)."""
    q = q.double()
    batch, heads, dim = q.shape
    group = heads // k_all.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, value_size = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((batch, heads), -math.inf, dtype=torch.float64, device=q.device)
    score_size = torch.zeros_like(lse)
    for b in range(batch):
        last = int(lengths[b])
        first = max(0, last - window) if window else 0
        if last == first:
            continue
        pages = tables[b].long()[: -(-last // page_size)]
        for h in range(heads):
            k, v = (x[pages, h // group].reshape(-1, dim)[first:last] for x in (k_all, v_all))
            s = (k @ q[b, h]) * scale
            p = torch.softmax(s, dim=0)
            lse[b, h] = torch.logsumexp(s, dim=0)
            out[b, h] = p @ v
            value_size[b, h] = p @ v.abs()
            score_size[b, h] = ((k.abs() @ q[b, h].abs()) * abs(scale)).max()
    return out, lse, value_size, score_size


def tables_for(lengths, page_size, num_pages, g, extra=0):
    """Block tables of distinct pages in no order; -1 behind each sequence's last."""
    used = [-(-n // page_size) for n in lengths]
    order = torch.randperm(num_pages, generator=g)
    assert sum(used) <= num_pages
    table = torch.full((len(lengths), max(max(used), 1) + extra), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    return table
