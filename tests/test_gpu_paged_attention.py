"""`paged_attention` against softmax attention in 64 bits over what the cache stands for."""

import math

import pytest
import torch

import chord_b200
from tests import attention_cases as A

pytestmark = pytest.mark.gpu


def make(device, lengths, heads, kv_heads, dim, page, bits, seed=0, spare=1):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-n // page) for n in lengths) + spare
    cache = chord_b200.kv_cache(pages, page, kv_heads, dim, dtype=torch.uint8 if bits == 8 else torch.bfloat16, device=device)
    A.fill(cache, torch.Generator(device=device).manual_seed(seed))
    table = A.tables_for(lengths, page, pages, g).to(device)
    q = (torch.randn((len(lengths), heads, dim), generator=g) * 1.5).to(torch.bfloat16).to(device)
    return q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=device)


def check(q, cache, table, lengths, out, lse=None, **options):
    """out: one rounding to BF16, P to 2^-16, the scores' additions; lse: the scores' additions."""
    want, want_lse, value_size, score_size = A.attention(q, *A.stored(cache), table, lengths, cache.page_size, **options)
    dim = q.shape[2]
    score = ((dim / 16 + 4) * A.SINGLE * score_size + 2.0 ** -20 * (1 + want_lse.abs().nan_to_num(posinf=0)))
    limit = A.HALF * want.abs() + (2.0 ** -16 + 2 * score[..., None]) * value_size * 1.01
    far = (out.double() - want).abs() - limit
    assert bool((far <= 0).all()), float(far.max())
    if lse is not None:
        empty = torch.isinf(want_lse)
        assert torch.equal(lse.double()[empty], want_lse[empty])
        assert bool(((lse.double() - want_lse).abs()[~empty] <= score[~empty]).all())


def run(q, cache, table, lengths, **options):
    lse = torch.full(q.shape[:2], float("nan"), device=q.device)
    out = chord_b200.paged_attention(q, cache, table, lengths, lse=lse, **options)
    chord_b200.check_status(q.device)
    return out, lse


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("heads,kv_heads,page,lengths", [
    (1, 1, 1, [1]), (8, 1, 16, [2, 16, 17, 0, 63, 64, 65]), (6, 2, 24, [500, 1, 0, 129]), (12, 1, 32, [300, 31]),
    (40, 2, 7, [200, 77]), (16, 16, 64, [128, 127, 129]), (9, 3, 100, [1500, 3]),
])
def test_small(device, heads, kv_heads, page, lengths, dim, bits):
    case = make(device, lengths, heads, kv_heads, dim, page, bits, seed=dim + len(lengths))
    out, lse = run(*case)
    check(*case, out, lse)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 64, 8), (64, 32, 1), (256, 8, 4), (128, 13, 13), (192, 20, 2)])
def test_long_and_ragged(device, dim, heads, kv_heads, bits):
    """Sequences that many CTAs share, beside short and empty ones; twice the same bits."""
    case = make(device, [20000, 1, 0, 333, 5001, 16], heads, kv_heads, dim, 16, bits, seed=heads)
    out, lse = run(*case)
    check(*case, out, lse)
    for _ in range(3):
        again, again_lse = run(*case)
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 100000])
def test_window(device, window, bits):
    case = make(device, [1, 64, 130, 1000, 0, 333], 8, 2, 128, 24, bits, seed=window)
    out, lse = run(*case, window=window)
    check(*case, out, lse, window=window)


def test_many_sequences(device):
    """More sequences than threads of a CTA, most of them empty."""
    lengths = [0] * 700
    for b in range(0, 700, 9):
        lengths[b] = 1 + b % 150
    case = make(device, lengths, 4, 2, 64, 16, 16, seed=5)
    out, lse = run(*case)
    check(*case, out, lse)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_scale(device, scale):
    case = make(device, [100, 700], 8, 1, 128, 16, 16, seed=3)
    out, lse = run(*case, scale=scale)
    check(*case, out, lse, scale=scale)


def test_peaked_scores(device):
    """Scores in the thousands: the running maximum moves all the time, and one token takes all."""
    q, cache, table, lengths = make(device, [2000, 64], 8, 2, 128, 16, 16, seed=9)
    q = q * 64
    out, lse = run(q, cache, table, lengths)
    check(q, cache, table, lengths, out, lse)


def test_garbage_behind_the_last_token(device):
    """NaN and infinities in unused places of the last page, in unused pages and in unused entries of the
    table change nothing."""
    q, cache, table, lengths = make(device, [37, 100], 8, 2, 128, 32, 16, seed=1, spare=2)
    want, _ = run(q, cache, table, lengths)
    used = torch.zeros((cache.num_pages, cache.page_size), dtype=torch.bool)
    for b, n in enumerate([37, 100]):
        for t in range(n):
            used[int(table[b, t // 32]), t % 32] = True
    free = (~used)[:, None, :, None].expand_as(cache.k).to(device)
    cache.k.masked_fill_(free, float("nan"))
    cache.v.masked_fill_(free, float("inf"))
    got, _ = run(q, cache, table, lengths)
    assert torch.equal(got, want)
    coded = make(device, [37, 100], 8, 2, 128, 32, 8, seed=1, spare=2)
    want, _ = run(*coded)
    free = (~used)[:, None, :].expand_as(coded[1].k_scale).to(device)
    coded[1].k_scale.masked_fill_(free, float("nan"))
    coded[1].v_scale.masked_fill_(free, float("inf"))
    got, _ = run(*coded)
    assert torch.equal(got, want)


def test_infinities_and_nan_in_the_tokens(device):
    q, cache, table, lengths = make(device, [90, 90, 90], 4, 1, 64, 16, 16, seed=2)
    q[0] = q[0].abs()
    cache.k[int(table[0, 1]), 0, 3] = float("-inf")      # score -inf: as if it were not there
    cache.v[int(table[1, 2]), 0, 5, 7] = float("nan")    # one dim of the output
    cache.k[int(table[2, 0]), 0, 0, 0] = float("nan")    # every output of the sequence
    out, lse = run(q, cache, table, lengths)
    k, v = A.stored(cache)
    keep = [t for t in range(90) if t != 19]
    pages = table[0].long()
    s = (k[pages, 0].reshape(-1, 64)[keep] @ q[0].double().t()) / 8.0
    want = torch.softmax(s, dim=0).t() @ v[pages, 0].reshape(-1, 64)[keep]
    assert bool(((out[0].double() - want).abs() <= A.HALF * want.abs() + 2.0 ** -13).all())
    assert torch.equal(torch.isnan(out[1]), (torch.arange(64, device=device) == 7).expand(4, 64))
    assert bool(torch.isnan(out[2]).all()) and bool(torch.isnan(lse[2]).all())
    assert bool(torch.isfinite(lse[:2]).all())


def test_all_scores_minus_infinity(device):
    """The first hundred tokens, then all of them."""
    q, cache, table, lengths = make(device, [150], 2, 1, 64, 16, 16, seed=2)
    q = q.abs()
    pages = table[0].long()
    cache.k[pages[:6]] = float("-inf")
    cache.k[pages[6], :, :4] = float("-inf")
    out, lse = run(q, cache, table, lengths)
    k, v = A.stored(cache)
    s = (k[pages, 0].reshape(-1, 64)[100:150] @ q[0].double().t()) / 8.0
    want = torch.softmax(s, dim=0).t() @ v[pages, 0].reshape(-1, 64)[100:150]
    assert bool(((out[0].double() - want).abs() <= A.HALF * want.abs() + 2.0 ** -13).all())
    cache.k.fill_(float("-inf"))
    out, lse = run(q, cache, table, lengths)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_shared_pages_strides_and_layouts(device):
    """Two sequences with common pages, queries inside a wider tensor, a table inside a wider one, and pages
    with the tokens before the heads."""
    g = torch.Generator(device=device).manual_seed(4)
    k, v = (torch.randn((9, 16, 2, 128), generator=g, device=device).to(torch.bfloat16).transpose(1, 2) for _ in range(2))
    cache = chord_b200.KVCache(k, v)
    wide = torch.randint(0, 9, (2, 12), dtype=torch.int32, device=device, generator=g)
    wide[:, 3:6] = torch.tensor([4, 1, 7], dtype=torch.int32)
    table = wide[:, 3:10]
    qkv = torch.randn((2, 12, 136), generator=g, device=device).to(torch.bfloat16)
    q = qkv[:, :8, :128]
    lengths = torch.tensor([100, 48], dtype=torch.int32, device=device)
    out, lse = run(q, cache, table, lengths)
    check(q, cache, table, lengths, out, lse)


def test_another_stream_and_a_graph(device):
    q, cache, table, lengths = make(device, [3000, 20], 16, 2, 128, 64, 8, seed=8)
    want, _ = run(q, cache, table, lengths)
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        got = chord_b200.paged_attention(q, cache, table, lengths)
    torch.cuda.current_stream(device).wait_stream(stream)
    assert torch.equal(got, want)
    locks = torch.zeros(1024, dtype=torch.int32, device=device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chord_b200.paged_attention(q, cache, table, lengths, locks=locks)
    lengths[0] = 1234      # lengths are read on the device, not fixed by the capture
    for _ in range(2):
        graph.replay()
        check(q, cache, table, lengths, out)
    assert bool((locks == 0).all())


def test_with_programmatic_launches(device):
    """Write and attend back to back with early launches: the attention sees what was written before it."""
    q, cache, table, lengths = make(device, [513, 70], 8, 2, 128, 16, 16, seed=6)
    k, v = (torch.randn((2, 2, 128), generator=torch.Generator().manual_seed(s)).to(torch.bfloat16).to(device) for s in (1, 2))
    slots = torch.tensor([int(table[0, 32]) * 16, int(table[1, 4]) * 16 + 5], dtype=torch.int32, device=device)
    chord_b200.set_option("pdl", 1)
    try:
        for i in range(20):
            chord_b200.cache_write(k * (i + 1), v * (i + 1), cache, slots)
            out, lse = chord_b200.paged_attention(q, cache, table, lengths), None
        check(q, cache, table, lengths, out)
    finally:
        chord_b200.set_option("pdl", 0)


def test_pages_and_lengths_outside(device):
    q, cache, table, lengths = make(device, [40, 40], 4, 1, 64, 16, 16, seed=7)
    want, _ = run(q, cache, table, lengths)
    bad = table.clone()
    bad[1, 1] = cache.num_pages
    out = chord_b200.paged_attention(q, cache, bad, lengths)
    assert torch.equal(out[0], want[0])
    with pytest.raises(RuntimeError, match="outside"):
        chord_b200.check_status(device)
    bad[1, 1] = -3
    chord_b200.paged_attention(q, cache, bad, lengths)
    with pytest.raises(RuntimeError, match="outside"):
        chord_b200.check_status(device)
    long = torch.tensor([48, 49], dtype=torch.int32, device=device)      # the table has three pages
    chord_b200.paged_attention(q, cache, table, long)
    with pytest.raises(RuntimeError, match="outside"):
        chord_b200.check_status(device)
    negative = torch.tensor([-5, 40], dtype=torch.int32, device=device)
    out = chord_b200.paged_attention(q, cache, table, negative)
    chord_b200.check_status(device)
    assert bool((out[0] == 0).all()) and torch.equal(out[1], want[1])


def test_parts_joined_by_lse(device):
    """Two halves of a sequence, joined with their lse, are the whole."""
    q, cache, table, lengths = make(device, [512], 8, 2, 128, 64, 16, seed=12)
    half = torch.tensor([256], dtype=torch.int32, device=device)
    whole, lse = run(q, cache, table, lengths)
    parts = [run(q, cache, t.contiguous(), half) for t in (table[:, :4], table[:, 4:])]
    top = torch.maximum(parts[0][1], parts[1][1])
    weights = [torch.exp(p[1] - top)[..., None] for p in parts]
    joined = sum(w * p[0].float() for w, p in zip(weights, parts)) / sum(weights)
    # three roundings to BF16 of values no larger than the parts'
    size = torch.maximum(parts[0][0].abs(), parts[1][0].abs()).float() + whole.abs().float()
    assert bool(((joined - whole.float()).abs() <= 2 * A.HALF * size + 1e-4).all())


def test_a_cache_past_four_gigabytes(device):
    q, cache, table, lengths = make(device, [100], 8, 8, 128, 64, 16, seed=3)
    pages = (5 << 30) // (8 * 128 * 64 * 2)
    far = chord_b200.kv_cache(pages, 64, 8, 128, device=device)
    for to, at in ((far.k, cache.k), (far.v, cache.v)):
        to[pages - 2:] = at[table[0].long()]
    want, _ = run(q, cache, table, lengths)
    got, _ = run(q, far, torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device=device), lengths)
    assert torch.equal(got, want)


def test_refusals(device):
    q, cache, table, lengths = make(device, [40, 40], 4, 2, 64, 16, 16)
    call = chord_b200.paged_attention
    with pytest.raises(TypeError, match="KVCache"):
        call(q, cache.k, table, lengths)
    with pytest.raises(TypeError, match="q must be"):
        call(q.float(), cache, table, lengths)
    with pytest.raises(ValueError, match="multiple of the cache"):
        call(q[:, :3], cache, table, lengths)
    with pytest.raises(ValueError, match="shape"):
        call(q[..., :32], cache, table, lengths)
    with pytest.raises(TypeError, match="block_tables"):
        call(q, cache, table.long(), lengths)
    with pytest.raises(ValueError, match="block_tables"):
        call(q, cache, table[:1], lengths)
    with pytest.raises(ValueError, match="lengths"):
        call(q, cache, table, lengths[:1])
    with pytest.raises(ValueError, match="window"):
        call(q, cache, table, lengths, window=0)
    with pytest.raises(ValueError, match="scale"):
        call(q, cache, table, lengths, scale=float("inf"))
    with pytest.raises(ValueError, match="lse"):
        call(q, cache, table, lengths, lse=torch.zeros((2, 3), device=device))
    with pytest.raises(RuntimeError, match="lock words"):
        call(q, cache, table, lengths, locks=torch.zeros(8, dtype=torch.int32, device=device))
    with pytest.raises(ValueError, match="outputs"):
        call(q, cache, table, lengths, outputs=q[:, :2])
    odd = chord_b200.kv_cache(2, 16, 2, 80, device=device)
    with pytest.raises(ValueError, match="head_dim"):
        call(torch.zeros((2, 4, 80), dtype=torch.bfloat16, device=device), odd, table, lengths)
    assert call(q[:0], cache, table[:0], lengths[:0]).shape == (0, 4, 64)
