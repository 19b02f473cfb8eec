"""One decoder layer of a model with 4-bit weights, a token at a time, on chord_b200.

    python examples/decode_layer.py [--batch B] [--steps S] [--bits 8|16]

Attention: qkv projection (gemv) -> norms, rotation and the 8-bit cache (qk_norm_rope_write) -> paged_attention
-> output projection (gemv).  Experts: a router (torch) -> gate_up -> SiLU*mul -> down, for a few tokens with
gemv on each token's own experts, for more through routing blocks (moe_align_block_size and indexed).  The
step is captured in a CUDA graph and replayed; block tables, lengths and slots change between replays.
Weights are random.  Prints the time of a step and how far the layer is from the same layer in FP32.
"""

import argparse
import dataclasses
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import chord_b200  # noqa: E402


@dataclasses.dataclass
class Shape:
    hidden: int = 1024
    heads: int = 16
    kv_heads: int = 2
    head_dim: int = 128
    experts: int = 16
    top_k: int = 4
    inter: int = 512
    page: int = 16
    max_tokens: int = 512     # of a sequence
    eps: float = 1e-6


FEW_TOKENS = 4  # up to here every token's experts are read for it alone
MAX_BATCH = 16  # rows of a gemv


def slots_for(tables: torch.Tensor, positions: torch.Tensor, page: int) -> torch.Tensor:
    """Where each sequence's token at its position is kept; nowhere (-1) past the last page of its table, so that
    a sequence that has outgrown its pages is reported by check_status and touches nothing."""
    pages = tables.shape[1]
    index = positions // page
    slots = tables.gather(1, index.clamp(0, pages - 1).long()[:, None])[:, 0] * page + positions % page
    return torch.where((index >= 0) & (index < pages), slots, -1).to(torch.int32)


def _check_sizes(shape: Shape, batch: int, steps: int) -> None:
    if not 1 <= batch <= MAX_BATCH:
        raise ValueError(f"batch must be from 1 to {MAX_BATCH}, got {batch}")
    if not 1 <= steps <= shape.max_tokens - 4:
        raise ValueError(f"steps must be from 1 to {shape.max_tokens - 4}, got {steps}")


def _packed(experts, n, k, g, keep):
    codes = torch.randint(0, 16, (experts, n, k), dtype=torch.int32, generator=g, device="cuda")
    scale = (torch.rand((experts, n, k // 32), generator=g, device="cuda") * 0.5 + 0.5) / (4.6 * k ** 0.5)
    scale = scale.to(torch.bfloat16)
    keep.append((codes.float() - 8) * scale.float().repeat_interleave(32, dim=2))
    return chord_b200.pack_w4a16(codes, scale)


class DecodeLayer:
    """The layer's weights, its cache and what a batch of sequences keeps between tokens."""

    def __init__(self, shape: Shape, batch: int, bits: int = 8, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        s = self.shape = shape
        self.batch = batch
        plain = []  # FP32 weights, for the comparison
        self.qkv = _packed(1, (s.heads + 2 * s.kv_heads) * s.head_dim, s.hidden, g, plain)
        self.out = _packed(1, s.hidden, s.heads * s.head_dim, g, plain)
        self.gate_up = _packed(s.experts, 2 * s.inter, s.hidden, g, plain)
        self.down = _packed(s.experts, s.hidden, s.inter, g, plain)
        self.plain = plain
        self.router = torch.randn((s.experts, s.hidden), generator=g, device="cuda").to(torch.bfloat16)
        self.q_weight, self.k_weight = ((torch.rand(s.head_dim, generator=g, device="cuda") + 0.5).to(torch.bfloat16)
                                        for _ in range(2))
        rate = 10000.0 ** (-torch.arange(0, s.head_dim, 2, device="cuda", dtype=torch.float64) / s.head_dim)
        angle = torch.arange(s.max_tokens, device="cuda", dtype=torch.float64)[:, None] * rate
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        pages = -(-s.max_tokens // s.page)
        self.cache = chord_b200.kv_cache(batch * pages, s.page, s.kv_heads, s.head_dim,
                                         dtype=torch.uint8 if bits == 8 else torch.bfloat16)
        # Pages are handed out in no order, as they come free in a server.
        self.tables = torch.randperm(batch * pages, generator=g, device="cuda").to(torch.int32).view(batch, pages)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.locks = torch.zeros(1024, dtype=torch.int32, device="cuda")

    def attention(self, x: torch.Tensor) -> torch.Tensor:
        s = self.shape
        positions = self.lengths.clone()
        slots = slots_for(self.tables, positions, s.page)
        qkv = chord_b200.gemv(x, self.qkv).view(self.batch, s.heads + 2 * s.kv_heads, s.head_dim)
        q, k, v = qkv.split([s.heads, s.kv_heads, s.kv_heads], dim=1)
        q = chord_b200.qk_norm_rope_write(q, k, v, self.q_weight, self.k_weight, self.cos_sin, positions, self.cache,
                                          slots, eps=s.eps)
        self.lengths += 1
        a = chord_b200.paged_attention(q, self.cache, self.tables, self.lengths, locks=self.locks)
        return chord_b200.gemv(a.view(self.batch, -1), self.out)

    def experts(self, x: torch.Tensor) -> torch.Tensor:
        s = self.shape
        scores, ids = torch.softmax(x.float() @ self.router.float().t() / s.hidden ** 0.5, dim=1).topk(s.top_k, dim=1)
        ids = ids.to(torch.int32)
        if self.batch <= FEW_TOKENS:
            h = chord_b200.silu_mul(chord_b200.gemv(x, self.gate_up, expert_ids=ids, top_k=s.top_k))
            y = chord_b200.gemv(h, self.down, expert_ids=ids)
        else:
            block_m = chord_b200.indexed_block_m(self.gate_up, self.batch, s.top_k)
            routing = chord_b200.moe_align_block_size(ids, block_m, s.experts)
            h = chord_b200.indexed(x, self.gate_up, *routing, s.top_k, block_m=block_m, locks=self.locks)
            h = chord_b200.silu_mul(h, sorted_ids=routing[0], num_tokens_padded=routing[2])
            y = chord_b200.indexed(h, self.down, *routing, 1, block_m=block_m, locks=self.locks)
        return (y.view(self.batch, s.top_k, s.hidden).float() * scores[:, :, None]).sum(dim=1).to(torch.bfloat16)

    def _norm(self, x: torch.Tensor) -> torch.Tensor:
        x = x.float()
        return (x * torch.rsqrt(x.pow(2).mean(dim=1, keepdim=True) + self.shape.eps)).to(torch.bfloat16)

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """One new token of each sequence, BF16 [batch, hidden]; batch at most 16."""
        x = x + self.attention(self._norm(x))
        return x + self.experts(self._norm(x))


class PlainLayer:
    """The same layer in FP32 on unpacked weights, with keys and values as they are."""

    def __init__(self, layer: DecodeLayer):
        self.layer, self.keys, self.values = layer, [], []

    def step(self, x: torch.Tensor) -> torch.Tensor:
        layer, s, x = self.layer, self.layer.shape, x.float()
        qkv_w, out_w, gate_up_w, down_w = layer.plain
        half = s.head_dim // 2
        cos, sin = layer.cos_sin[len(self.keys)].split(half)

        def norm(v, w=1.0):
            return v * torch.rsqrt(v.pow(2).mean(dim=-1, keepdim=True) + s.eps) * w

        def turn(v):
            a, b = v[..., :half], v[..., half:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)

        qkv = (norm(x) @ qkv_w[0].t()).view(layer.batch, -1, s.head_dim)
        q, k, v = qkv.split([s.heads, s.kv_heads, s.kv_heads], dim=1)
        q, k = turn(norm(q, layer.q_weight.float())), turn(norm(k, layer.k_weight.float()))
        self.keys.append(k)
        self.values.append(v)
        group = s.heads // s.kv_heads
        keys, values = (torch.stack(t, dim=2).repeat_interleave(group, dim=1) for t in (self.keys, self.values))
        p = torch.softmax((keys @ q[..., None])[..., 0] * s.head_dim ** -0.5, dim=-1)
        x = x + (p[:, :, None] @ values)[:, :, 0].reshape(layer.batch, -1) @ out_w[0].t()
        h = norm(x)
        scores, ids = torch.softmax(h @ layer.router.float().t() / s.hidden ** 0.5, dim=1).topk(s.top_k, dim=1)
        y = torch.zeros_like(x)
        for b in range(layer.batch):
            for j in range(s.top_k):
                gate, up = (gate_up_w[ids[b, j]] @ h[b]).chunk(2)
                y[b] += scores[b, j] * (down_w[ids[b, j]] @ (torch.nn.functional.silu(gate) * up))
        return x + y


def compare(shape: Shape, batch: int, steps: int, bits: int, seed: int = 0) -> float:
    """Relative distance (2-norm) of the layer's outputs from the plain layer's, over all steps."""
    _check_sizes(shape, batch, steps)
    layer = DecodeLayer(shape, batch, bits, seed)
    plain = PlainLayer(layer)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    off = size = 0.0
    for _ in range(steps):
        x = torch.randn((batch, shape.hidden), generator=g, device="cuda").to(torch.bfloat16)
        want = plain.step(x)
        off += float((layer.step(x).float() - want).pow(2).sum())
        size += float(want.pow(2).sum())
    chord_b200.check_status()
    return (off / size) ** 0.5


def time_step(shape: Shape, batch: int, steps: int, bits: int) -> float:
    """Microseconds of a step, replayed from a CUDA graph."""
    _check_sizes(shape, batch, steps)
    layer = DecodeLayer(shape, batch, bits)
    x = torch.randn((batch, shape.hidden), device="cuda").to(torch.bfloat16)
    for _ in range(2):
        layer.step(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(x)
    layer.lengths.fill_(shape.max_tokens - steps - 4)
    graph.replay()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(steps):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    chord_b200.check_status()
    return begin.elapsed_time(end) * 1e3 / steps


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--bits", type=int, default=8, choices=[8, 16])
    a = ap.parse_args()
    try:
        _check_sizes(Shape(), a.batch, a.steps)
    except ValueError as e:
        ap.error(str(e))
    print(f"relative distance from FP32 over {a.steps} tokens: {compare(Shape(), a.batch, a.steps, a.bits):.2e}")
    print(f"a step: {time_step(Shape(), a.batch, a.steps, a.bits):.1f} us")


if __name__ == "__main__":
    main()
