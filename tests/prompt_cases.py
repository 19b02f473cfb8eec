"""Inputs and 64-bit plain forms of `prompt_attention`, `shared_prefix_attention` and shaped scores, with the
limits that their arithmetic sets, shared by the tests.  Written from the definitions."""

from __future__ import annotations

import math

import torch

import chord_b200
from tests import attention_cases as A


def rows_of(cache, table, count):
    """float64 keys and values [count, kv_heads, dim] that a sequence's first tokens stand for."""
    at = torch.arange(count, device=table.device)
    pages = table.long()[at // cache.page_size]
    k, v = A.stored(cache)
    return k[pages, :, at % cache.page_size], v[pages, :, at % cache.page_size]


def attend(q, k, v, position, low, high, *, scale=None, cap=None, slopes=None):
    """Query tokens q [n, heads, dim], the i-th at position[i] and seeing tokens low[i] to high[i] of k and v
    [tokens, kv_heads, dim], which others may be anything.  float64 out, lse, sizes of the values' terms,
    and how far a score may be off."""
    n, heads, dim = q.shape
    q, group, scale = q.double(), heads // k.shape[1], dim ** -0.5 if scale is None else scale
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device=q.device)
    error = torch.zeros_like(lse)
    for i in range(n):
        a, b = max(0, int(low[i])), int(high[i])
        if b <= a:
            continue
        keys, values = (x[a:b].repeat_interleave(group, dim=1) for x in (k, v))  # [tokens, heads, dim]
        s = torch.einsum("thd,hd->ht", keys, q[i]) * scale
        off = (dim / 16 + 4) * A.SINGLE * torch.einsum("thd,hd->ht", keys.abs(), q[i].abs()) * abs(scale)
        if cap:
            s = cap * torch.tanh(s / cap)
            off = off + 2.0 ** -21 * cap
        if slopes is not None:
            lean = slopes.double()[:, None] * (torch.arange(a, b, device=q.device) - int(position[i])).abs()
            s = s - lean
            off = off + 4 * A.SINGLE * lean
        p = torch.softmax(s, dim=1)
        lse[i] = torch.logsumexp(s, dim=1)
        out[i] = torch.einsum("ht,thd->hd", p, values)
        size[i] = torch.einsum("ht,thd->hd", p, values.abs())
        error[i] = (off + 2.0 ** -22 * s.abs()).amax(dim=1)  # (and the exponential's argument is rounded)
    return out, lse, size, error


def close(got, want, *, weights=A.HALF):
    """out: one rounding to BF16, each weight's rounding (``weights``, relative) and what its score is off by, twice
    since the weights' sum is off as well; lse: the scores' error, and FP32 logarithms.  Sums over thousands of
    terms in FP32 stay below a hundredth of the first two."""
    out, lse, size, error = want
    score = error + 2.0 ** -20 * (1 + lse.abs().nan_to_num(posinf=0))
    limit = A.HALF * out.abs() + (1.01 * weights + 2 * score[..., None]) * size * 1.01 + 1e-30
    far = (got[0].double() - out).abs() - limit
    assert bool((far <= 0).all()), (float(far.max()), (far > 0).nonzero()[:4].tolist())
    empty = torch.isinf(lse)
    assert torch.equal(got[1].double()[empty], lse[empty])
    assert bool(((got[1].double() - lse).abs()[~empty] <= score[~empty]).all())


class Prompt:
    """A ragged batch: (past, new) tokens of each sequence, in a cache of its own."""

    def __init__(self, device, sequences, heads, kv_heads, dim, page, bits, seed=0, spare=1, rows_behind=0):
        g = torch.Generator().manual_seed(seed)
        self.past, self.new = [a for a, _ in sequences], [b for _, b in sequences]
        total = [a + b for a, b in sequences]
        pages = sum(-(-n // page) for n in total) + spare
        self.cache = chord_b200.kv_cache(pages, page, kv_heads, dim, dtype=torch.uint8 if bits == 8 else torch.bfloat16, device=device)
        A.fill(self.cache, torch.Generator(device=device).manual_seed(seed))
        self.table = A.tables_for(total, page, pages, g).to(device)
        self.lengths = torch.tensor(total, dtype=torch.int32, device=device)
        self.ends = torch.tensor([0] + self.new).cumsum(0).tolist()
        self.offsets = torch.tensor(self.ends, dtype=torch.int32, device=device)
        self.q = (torch.randn((self.ends[-1] + rows_behind, heads, dim), generator=g) * 1.5).to(torch.bfloat16).to(device)
        self.slopes = (2.0 ** (-8 * torch.arange(1, heads + 1) / heads)).to(device)

    def run(self, **options):
        lse = torch.full(self.q.shape[:2], float("nan"), device=self.q.device)
        out = chord_b200.prompt_attention(self.q, self.cache, self.table, self.lengths, self.offsets, lse=lse, **options)
        chord_b200.check_status(self.q.device)
        return out, lse

    def want(self, *, window=None, starts=None, prefixes=None, **options):
        parts = []
        for b, n in enumerate(self.new):
            length = self.past[b] + n
            position = torch.arange(length - n, length)
            low = (position + 1 - window).clamp(min=0) if window else torch.zeros_like(position)
            high = position + 1
            if starts is not None:
                low = torch.maximum(low, starts[self.ends[b]:self.ends[b + 1]].cpu().long())
            if prefixes is not None:
                high = high.clamp(min=min(int(prefixes[b]), length))
            k, v = rows_of(self.cache, self.table[b], length)
            parts.append(attend(self.q[self.ends[b]:self.ends[b + 1]], k, v, position, low, high, **options))
        return tuple(torch.cat(x) for x in zip(*parts))

    def check(self, got=None, **options):
        got = self.run(**options) if got is None else got
        rows = self.ends[-1]
        close([x[:rows] for x in got], self.want(**options))
        return got
