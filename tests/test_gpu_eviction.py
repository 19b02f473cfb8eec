"""`attention_weights` and `cache_evict` against their definitions in 64 bits."""

import math

import pytest
import torch

import chord_b200
from tests import attention_cases as A
from tests.prompt_cases import attend, rows_of

pytestmark = pytest.mark.gpu


def make(device, lengths, kv_heads, dim, page, bits, seed=0, spare=1, more=()):
    """A cache with the sequences' tables and, of further lengths, tables of other pages."""
    g = torch.Generator().manual_seed(seed)
    every = list(lengths) + list(more)
    pages = sum(-(-n // page) for n in every) + spare
    cache = chord_b200.kv_cache(pages, page, kv_heads, dim, dtype=torch.uint8 if bits == 8 else torch.bfloat16, device=device)
    A.fill(cache, torch.Generator(device=device).manual_seed(seed))
    table = A.tables_for(every, page, pages, g).to(device)
    return cache, table[:len(lengths)].contiguous(), table[len(lengths):].contiguous(), torch.tensor(lengths, dtype=torch.int32, device=device)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("heads,kv_heads,page,lengths", [
    (1, 1, 1, [1]), (8, 1, 16, [2, 63, 64, 65, 0]), (6, 2, 24, [500, 1]), (40, 2, 7, [200, 77]), (9, 3, 100, [1500, 3]),
])
@pytest.mark.parametrize("shape", ["plain", "cap", "all"])
def test_weights(device, shape, heads, kv_heads, page, lengths, dim, bits):
    cache, table, _, n = make(device, lengths, kv_heads, dim, page, bits, seed=dim)
    g = torch.Generator().manual_seed(7)
    q = (torch.randn((len(lengths), heads, dim), generator=g) * 1.5).to(torch.bfloat16).to(device)
    slopes = (2.0 ** (-8 * torch.arange(1, heads + 1) / heads)).to(device)
    options = {"plain": {}, "cap": dict(cap=5.0), "all": dict(cap=20.0, slopes=slopes, window=40, scale=0.2)}[shape]
    lse = torch.empty((len(lengths), heads), device=device)
    chord_b200.paged_attention(q, cache, table, n, lse=lse, **options)
    got = chord_b200.attention_weights(q, cache, table, n, lse, **options)
    chord_b200.check_status(device)
    width = table.shape[1] * page
    assert got.shape == (len(lengths), kv_heads, width)
    again = chord_b200.attention_weights(q, cache, table, n, lse, weights=torch.ones((len(lengths), kv_heads, width + 3), device=device),
                                         **options)
    assert torch.equal(again[:, :, :width], got + 1) and bool((again[:, :, width:] == 1).all())
    window = options.pop("window", None)
    for b, length in enumerate(lengths):
        low = max(0, length - window) if window else 0
        k, _ = rows_of(cache, table[b], length)
        _, _, _, error = attend(q[b:b + 1], k, k, [length - 1], [low], [length], **options)
        s = torch.einsum("thd,hd->ht", k.repeat_interleave(heads // kv_heads, dim=1), q[b].double()) * options.get("scale", dim ** -0.5)
        if "cap" in options:
            s = options["cap"] * torch.tanh(s / options["cap"])
        if "slopes" in options:
            s = s - slopes.double()[:, None] * (length - 1 - torch.arange(length, device=device))
        p = torch.exp(s - lse[b].double()[:, None])
        p[:, :low] = 0
        want = p.view(kv_heads, heads // kv_heads, length).sum(dim=1)
        # a score's error, the sum's that was given and the exponential's, relative
        off = (p * (2 * error[0] + 2.0 ** -20 * (1 + lse[b].double().abs()))[:, None].nan_to_num()).view(kv_heads, heads // kv_heads, length).sum(dim=1)
        assert bool(((got[b, :, :length].double() - want).abs() <= off + 1e-30).all())
        assert bool((got[b, :, length:] == 0).all()) and bool((got[b, :, :low] == 0).all())


def test_weights_of_sequences_that_see_nothing(device):
    cache, table, _, n = make(device, [40, 0], 2, 64, 16, 16)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=device)
    lse = torch.full((2, 4), -math.inf, device=device)
    assert bool((chord_b200.attention_weights(q, cache, table, n, lse) == 0).all())
    chord_b200.check_status(device)
    short = torch.zeros((2, 2, 30), device=device)
    chord_b200.attention_weights(q, cache, table, n, torch.zeros_like(lse), weights=short)
    assert bool((short[0] == 2).all()) and bool((short[1] == 0).all())
    with pytest.raises(RuntimeError, match="index"):
        chord_b200.check_status(device)


def kept_tokens(weights, length, keep, first, recent):
    """By the definition: sorted by (not held, weight downwards, place)."""
    if length <= keep:
        return list(range(length))
    held = lambda i: i < first or i >= length - recent
    key = lambda i: (not held(i), -(math.inf if math.isnan(weights[i]) else weights[i]) if not held(i) else 0,
                     not math.isnan(weights[i]), i)
    return sorted(sorted(range(length), key=key)[:keep])


def check_eviction(device, lengths, keep, first, recent, kv_heads, dim, page, bits, apart, seed=0, kind="random", wide=0):
    cache, table, other, n = make(device, lengths, kv_heads, dim, page, bits, seed=seed,
                                  more=[min(keep, x) for x in lengths] if apart else ())
    g = torch.Generator().manual_seed(seed)
    width = max(table.shape[1] * page, 1) + wide
    weights = torch.rand((len(lengths), kv_heads, width), generator=g) ** 4
    if kind == "equal":
        weights = torch.randint(0, 3, weights.shape, generator=g).float()
    elif kind == "zeros":
        weights = torch.where(torch.rand(weights.shape, generator=g) < 0.9, 0.0, weights)
        weights[torch.rand(weights.shape, generator=g) < 0.3] *= -1  # (minus zero among them)
    elif kind == "odd":
        weights[torch.rand(weights.shape, generator=g) < 0.1] = math.nan
        weights[torch.rand(weights.shape, generator=g) < 0.1] = math.inf
        weights[torch.rand(weights.shape, generator=g) < 0.1] = -math.inf
    before = [x.clone() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale) if x is not None]
    given = weights.to(device)
    got_lengths, got_weights = chord_b200.cache_evict(cache, table, n, given, keep, first=first, recent=recent,
                                                      new_tables=other if apart else None)
    chord_b200.check_status(device)
    assert torch.equal(given.cpu().nan_to_num(7), weights.nan_to_num(7))
    want = [x.clone() for x in before]
    want_weights = torch.zeros((len(lengths), kv_heads, max(width, keep)))
    for b, length in enumerate(lengths):
        for h in range(kv_heads):
            kept = torch.tensor(kept_tokens(weights[b, h].tolist(), length, keep, first, recent), dtype=torch.int64)
            want_weights[b, h, :len(kept)] = weights[b, h, kept]
            place, source = torch.arange(len(kept), device=device), kept.to(device)
            to = (other if apart else table)[b].long()
            for x, old in zip(want, before):
                x[to[place // page], h, place % page] = old[table[b].long()[source // page], h, source % page]
    assert got_lengths.tolist() == [min(x, keep) for x in lengths]
    assert torch.equal(got_weights.cpu().nan_to_num(7), want_weights.nan_to_num(7))
    for x, y in zip(want, (x for x in (cache.k, cache.v, cache.k_scale, cache.v_scale) if x is not None)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("apart", [True, False])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("lengths,keep,first,recent,kv_heads,dim,page", [
    ([1], 1, 0, 0, 1, 16, 1), ([2, 0, 5], 1, 0, 1, 2, 64, 4), ([300, 17, 0, 301], 100, 4, 16, 3, 96, 24),
    ([1000, 999], 998, 0, 0, 2, 128, 16), ([5000, 100], 1025, 7, 500, 2, 48, 100), ([700], 64, 32, 32, 1, 256, 64),
    ([2049, 2048, 2047], 2047, 1, 1, 1, 80, 7),
])
def test_eviction(device, lengths, keep, first, recent, kv_heads, dim, page, bits, apart):
    check_eviction(device, lengths, keep, first, recent, kv_heads, dim, page, bits, apart, seed=keep)


@pytest.mark.parametrize("apart", [True, False])
@pytest.mark.parametrize("kind", ["equal", "zeros", "odd"])
def test_ties_and_odd_weights(device, kind, apart):
    check_eviction(device, [900, 300, 4100], 257, 2, 9, 3, 64, 16, 16, apart, kind=kind, wide=5)
    check_eviction(device, [900, 300, 4100], 257, 0, 0, 3, 64, 16, 8, apart, kind=kind)


@pytest.mark.parametrize("kind", ["random", "zeros"])
def test_more_weights_than_shared_memory_holds(device, kind):
    check_eviction(device, [60000, 41000], 20000, 4, 64, 1, 16, 64, 16, False, kind=kind)


def test_room_behind_the_sequences(device):
    """Fewer tokens than are to be kept, and weights narrower than keep."""
    cache, table, _, n = make(device, [10, 3], 2, 64, 16, 16)
    weights = torch.rand((2, 2, 12), device=device)
    lengths, kept = chord_b200.cache_evict(cache, table, n, weights, 40)
    assert lengths.tolist() == [10, 3] and kept.shape == (2, 2, 40)
    assert torch.equal(kept[0, :, :10], weights[0, :, :10]) and bool((kept[0, :, 10:] == 0).all()) and bool((kept[1, :, 3:] == 0).all())


def test_bad_pages_are_reported(device):
    for apart in (True, False):
        cache, table, other, n = make(device, [100, 60], 2, 64, 16, 16, more=[50, 50])
        table[0, 1] = 5000
        chord_b200.cache_evict(cache, table, n, torch.rand((2, 2, 112), device=device), 50, first=30, new_tables=other if apart else None)
        with pytest.raises(RuntimeError, match="index"):
            chord_b200.check_status(device)
    cache, table, _, n = make(device, [100], 2, 64, 16, 16)
    chord_b200.cache_evict(cache, table, n, torch.rand((1, 2, 50), device=device), 30)
    with pytest.raises(RuntimeError, match="index"):
        chord_b200.check_status(device)


def test_a_served_sequence(device):
    """Prompt, tokens with their weights gathered, eviction, further tokens, replayed from one graph."""
    page, heads, kv_heads, dim, keep = 16, 8, 2, 64, 48
    g = torch.Generator(device=device).manual_seed(1)
    cache = chord_b200.kv_cache(32, page, kv_heads, dim, device=device)
    table = torch.randperm(32, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(2, 16).to(device)
    new = lambda *shape: torch.randn(shape, generator=g, device=device).to(torch.bfloat16)
    slots = lambda b, at: (table[b, at // page] * page + at % page).to(torch.int32)
    prompt = torch.tensor([70, 41])
    at = [torch.arange(int(n), device=device) for n in prompt]
    chord_b200.cache_write(new(111, kv_heads, dim), new(111, kv_heads, dim), cache, torch.cat([slots(b, a) for b, a in enumerate(at)]))
    lengths = prompt.to(torch.int32).to(device)
    offsets = torch.tensor([0, 70, 111], dtype=torch.int32, device=device)
    assert torch.isfinite(chord_b200.prompt_attention(new(111, heads, dim), cache, table, lengths, offsets).float()).all()
    q, k, v = new(2, heads, dim), new(2, kv_heads, dim), new(2, kv_heads, dim)
    weights = torch.zeros((2, kv_heads, 256), device=device)
    lse, locks = torch.empty((2, heads), device=device), torch.zeros(1024, dtype=torch.int32, device=device)
    out = torch.empty_like(q)

    def step():
        where = lengths.clone()
        chord_b200.cache_write(k, v, cache, (table.gather(1, (where // page)[:, None].long())[:, 0] * page + where % page).to(torch.int32))
        lengths.add_(1)
        chord_b200.paged_attention(q, cache, table, lengths, lse=lse, outputs=out, locks=locks)
        chord_b200.attention_weights(q, cache, table, lengths, lse, weights=weights)
        shorter, kept = chord_b200.cache_evict(cache, table, lengths, weights, keep, first=2, recent=8)
        lengths.copy_(shorter)
        weights.copy_(kept)

    step()
    torch.cuda.synchronize()
    chord_b200.check_status(device)
    assert lengths.tolist() == [48, 42]
    graph = torch.cuda.CUDAGraph()
    state = [x.clone() for x in (cache.k, cache.v, lengths, weights)]
    with torch.cuda.graph(graph):
        step()
    for x, y in zip((cache.k, cache.v, lengths, weights), state):
        x.copy_(y)
    for _ in range(9):
        graph.replay()
    torch.cuda.synchronize()
    chord_b200.check_status(device)
    by_graph = [x.clone() for x in (cache.k, cache.v, lengths, weights, out)]
    for x, y in zip((cache.k, cache.v, lengths, weights), state):
        x.copy_(y)
    for _ in range(9):
        step()
    for x, y in zip((cache.k, cache.v, lengths, weights, out), by_graph):
        assert torch.equal(x, y)
    assert lengths.tolist() == [48, 48]
