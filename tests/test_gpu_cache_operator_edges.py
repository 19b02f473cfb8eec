"""The operators over the cache at the edges of what they take: rows of other widths, lengths that are none, budgets beyond any
sequence, tables that name a page twice, calls on several streams at once."""

import math

import pytest
import torch

import chord_b200
from tests import attention_cases as A
from tests.prompt_cases import Prompt, close
from tests.test_gpu_eviction import check_eviction

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [16, 48, 80, 208])
def test_rows_of_other_widths(device, dim, bits, apart):
    check_eviction(device, [90, 7, 300], 41, 3, 5, 2, dim, 24, bits, apart, seed=dim)


def test_a_budget_beyond_any_sequence(device):
    cache = chord_b200.kv_cache(9, 16, 2, 64, device=device)
    A.fill(cache, torch.Generator(device=device).manual_seed(1))
    table = torch.arange(8, dtype=torch.int32, device=device).reshape(2, 4)
    other = torch.full((2, 4), 8, dtype=torch.int32, device=device)
    weights = torch.rand((2, 2, 50), device=device)
    before = cache.k.clone()
    lengths, held = chord_b200.cache_evict(cache, table, torch.tensor([50, 1], dtype=torch.int32, device=device), weights, 1 << 20)
    assert lengths.tolist() == [50, 1] and held.shape == (2, 2, 1 << 20) and torch.equal(cache.k, before)
    assert torch.equal(held[0, :, :50], weights[0]) and torch.equal(held[1, :, :1], weights[1, :, :1])
    assert float(held[0, :, 50:].abs().sum() + held[1, :, 1:].abs().sum()) == 0.0
    chord_b200.cache_evict(cache, table, torch.tensor([0, 1], dtype=torch.int32, device=device), weights, 1 << 20, new_tables=other)
    assert torch.equal(cache.k[8, :, 0], cache.k[4, :, 0]) and torch.equal(cache.k[:8], before[:8]) and torch.equal(cache.k[8, :, 1:], before[8, :, 1:])
    chord_b200.check_status(device)


@pytest.mark.parametrize("length", [-1, -2**31])
def test_lengths_below_zero_are_none(device, length):
    case = Prompt(device, [(0, 40), (30, 20)], 4, 2, 64, 16, 16, seed=3)
    zero, below = case.lengths.clone(), case.lengths.clone()
    zero[1], below[1] = 0, length
    q, lse = case.q[:2], torch.zeros((2, 4), device=device)
    groups, one = torch.tensor([0, 2], dtype=torch.int32, device=device), case.table[:1].contiguous()
    got = []
    for lengths in (zero, below):
        case.lengths = lengths
        out = [*case.run(), *case.run(window=7), *case.run(prefixes=torch.tensor([5, int(lengths[1])], dtype=torch.int32, device=device))]
        lse = torch.zeros((2, 4), device=device)
        out += [chord_b200.paged_attention(q, case.cache, case.table, lengths, cap=9.0, lse=lse), lse]
        out += [chord_b200.attention_weights(q, case.cache, case.table, lengths, lse, cap=9.0)]
        out += [chord_b200.shared_prefix_attention(q, case.cache, one, lengths[1:].contiguous(), groups, case.table, lengths)]
        out += list(chord_b200.cache_evict(case.cache, case.table, lengths, out[-2], 64))
        chord_b200.check_status(device)
        got.append(out)
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert bool((got[0][1][40:] == -math.inf).all()) and got[0][-2].tolist() == [40, 0]


@pytest.mark.parametrize("bits", [16, 8])
def test_a_page_named_twice(device, bits):
    """Readers take a table as it is: a sequence that holds one page several times, and two that share theirs."""
    case = Prompt(device, [(20, 28), (10, 38)], 6, 3, 128, 16, bits, seed=7)
    case.table[0, 2] = case.table[0, 0]
    case.table[1] = case.table[0]
    case.check()


def test_streams_at_once(device):
    cases = [Prompt(device, [(50 * i, 300), (700, 41)], 8, 2, 128, 16, 16 if i % 2 else 8, seed=i) for i in range(4)]
    want = [(*case.run(), *case.run(cap=20.0)) for case in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(5):
        for case, stream, results in zip(cases, streams, got):
            with torch.cuda.stream(stream):
                for cap in (None, 20.0):
                    lse = torch.zeros(case.q.shape[:2], device=device)
                    results.append(chord_b200.prompt_attention(case.q, case.cache, case.table, case.lengths, case.offsets, cap=cap, lse=lse))
                    results.append(lse)
    torch.cuda.synchronize()
    chord_b200.check_status(device)
    for results, expected in zip(got, want):
        for i, x in enumerate(results):
            assert torch.equal(x, expected[i % 4])


@pytest.mark.parametrize("bits", [16, 8])
def test_offsets_beyond_32_bits(device, bits):
    """The same pages at the end of a cache of more than 2^32 elements: the same bits."""
    case = Prompt(device, [(100, 60), (0, 90)], 16, 8, 128, 16, bits, seed=13)
    small, used = case.cache, case.cache.num_pages
    pages = 2**32 // (8 * 16 * 128) + used
    large = chord_b200.kv_cache(pages, 16, 8, 128, dtype=torch.uint8 if bits == 8 else torch.bfloat16, device=device)
    parts = lambda cache: [x for x in (cache.k, cache.v, cache.k_scale, cache.v_scale) if x is not None]  # noqa: E731
    for to, of in zip(parts(large), parts(small)):
        to[-used:] = of
    table, far = case.table.clamp(min=0), case.table.clamp(min=0) + (pages - used)
    lengths, groups, one = case.lengths, torch.tensor([0, 2], dtype=torch.int32, device=device), torch.tensor([160], dtype=torch.int32, device=device)
    got = []
    for cache, at in ((small, table), (large, far)):
        out = [chord_b200.prompt_attention(case.q, cache, at, lengths, case.offsets, cap=cap) for cap in (None, 9.0)]
        lse = torch.zeros((2, 16), device=device)
        out += [chord_b200.paged_attention(case.q[:2], cache, at, lengths, slopes=torch.ones(16, device=device), lse=lse)]
        out += [chord_b200.attention_weights(case.q[:2], cache, at, lengths, lse)]
        out += [chord_b200.shared_prefix_attention(case.q[:2], cache, at[:1].contiguous(), one, groups, at, lengths)]
        out += list(chord_b200.cache_evict(cache, at, lengths, out[3], 50, first=2, recent=9))
        chord_b200.check_status(device)
        got.append(out + [x[-used:] for x in parts(cache)])
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
def test_few_tokens_over_codes(device, dim):
    """Rows that see few tokens do not average the rounding of weights: two BF16 numbers each, off by 2^-16, and sums of
    at most 512 terms in FP32, each of which may be cut off at 2^-23 of the sum, in the result and in the weights' sum: 2^-13."""
    case = Prompt(device, [(0, 40), (3, 200), (150, 60), (0, 1)], 8, 2, dim, 16, 8, seed=31)
    close(case.run(), case.want(), weights=2.0 ** -16 + 2.0 ** -13)
    close(case.run(window=3, cap=8.0), case.want(window=3, cap=8.0), weights=2.0 ** -16 + 2.0 ** -13)
