"""`shared_prefix_attention`, and `paged_attention` with shaped scores, against 64 bits."""

import math

import pytest
import torch

import chord_b200
from tests import attention_cases as A
from tests.prompt_cases import attend, close, rows_of

pytestmark = pytest.mark.gpu


class Shared:
    """Groups of (prefix length, own lengths)."""

    def __init__(self, device, groups, heads, kv_heads, dim, page, bits, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.prefix = [p for p, _ in groups]
        self.own = [n for _, own in groups for n in own]
        self.group = [i for i, (_, own) in enumerate(groups) for _ in own]
        pages = sum(-(-n // page) for n in self.prefix + self.own) + 1
        self.cache = chord_b200.kv_cache(pages, page, kv_heads, dim, dtype=torch.uint8 if bits == 8 else torch.bfloat16, device=device)
        A.fill(self.cache, torch.Generator(device=device).manual_seed(seed))
        both = A.tables_for(self.prefix + self.own, page, pages, g).to(device)
        self.prefix_table, self.table = both[:len(groups)].contiguous(), both[len(groups):]
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
        self.prefix_lengths, self.lengths = ints(self.prefix), ints(self.own)
        self.offsets = ints([0] + torch.tensor([len(own) for _, own in groups]).cumsum(0).tolist())
        self.q = (torch.randn((len(self.own), heads, dim), generator=g) * 1.5).to(torch.bfloat16).to(device)
        self.slopes = (2.0 ** (-8 * torch.arange(1, heads + 1) / heads)).to(device)

    def run(self, **options):
        lse = torch.full(self.q.shape[:2], float("nan"), device=self.q.device)
        out = chord_b200.shared_prefix_attention(self.q, self.cache, self.prefix_table, self.prefix_lengths, self.offsets,
                                                 self.table, self.lengths, lse=lse, **options)
        chord_b200.check_status(self.q.device)
        return out, lse

    def check(self, *, window=None, **options):
        got = self.run(window=window, **options)
        parts = []
        for b, n in enumerate(self.own):
            p = self.prefix[self.group[b]]
            kv = [torch.cat(x) for x in zip(rows_of(self.cache, self.prefix_table[self.group[b]], p), rows_of(self.cache, self.table[b], n))]
            last = p + n
            parts.append(attend(self.q[b:b + 1], *kv, [last - 1], [last - window if window else 0], [last], **options))
        close(got, tuple(torch.cat(x) for x in zip(*parts)))
        return got


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("heads,kv_heads,page,groups", [
    (1, 1, 1, [(1, [1])]), (8, 1, 16, [(100, [3, 0, 40]), (0, [5, 0]), (64, [0])]), (6, 2, 24, [(333, [1] * 70), (1, [2])]),
    (40, 2, 7, [(130, [9, 300])]), (8, 8, 32, [(257, list(range(150)))]),
])
def test_small(device, heads, kv_heads, page, groups, dim, bits):
    Shared(device, groups, heads, kv_heads, dim, page, bits, seed=dim).check()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 16, 2), (64, 8, 8), (256, 4, 2)])
def test_long_prefixes(device, dim, heads, kv_heads, bits):
    case = Shared(device, [(20000, [30, 0, 200]), (3000, [1] * 33)], heads, kv_heads, dim, 64, bits, seed=dim)
    out, lse = case.check()
    for _ in range(3):
        again, again_lse = case.run()
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("shape", ["window", "narrow", "cap", "slopes", "all"])
def test_shaped(device, shape, bits):
    case = Shared(device, [(300, [70, 0, 10, 500]), (90, [1, 2])], 8, 2, 128, 16, bits, seed=4)
    case.check(**{"window": dict(window=100), "narrow": dict(window=3), "cap": dict(cap=5.0), "slopes": dict(slopes=case.slopes),
                  "all": dict(cap=20.0, slopes=case.slopes, window=200, scale=0.2)}[shape])


def test_equals_the_sequences_as_a_whole(device):
    """The same tokens in one table: both operators, to the rounding of the prefix's weights."""
    case = Shared(device, [(640, [30, 100, 64])], 8, 2, 128, 32, 16, seed=8)
    whole = torch.cat([case.prefix_table[:, :20].expand(3, 20), case.table], dim=1).contiguous()
    lse = torch.empty((3, 8), device=device)
    want = chord_b200.paged_attention(case.q, case.cache, whole, case.lengths + 640, lse=lse)
    out, got_lse = case.run()
    assert bool(((out.float() - want.float()).abs() <= 2.0 ** -8 * (want.float().abs() * 2 + 3)).all())
    assert torch.allclose(got_lse, lse, atol=1e-4)


def test_values_of_others_change_nothing(device):
    case = Shared(device, [(100, [20, 30]), (200, [5])], 4, 1, 128, 16, 16, seed=6)
    clean = case.run()
    for x in (case.cache.k, case.cache.v):
        x[int(case.table[1, 1])] = math.nan                                # of the second sequence alone
        x[int(case.prefix_table[1, 12]), :, 8:] = math.inf                 # behind the second prefix
    out, lse = case.run()
    for b in (0, 2):
        assert torch.equal(out[b], clean[0][b]) and torch.equal(lse[b], clean[1][b])
    assert bool(torch.isnan(out[1].float()).all())


def test_in_a_graph(device):
    case = Shared(device, [(1000, [20, 30]), (200, [5])], 16, 4, 128, 16, 16, seed=6)
    locks, out = torch.zeros(1024, dtype=torch.int32, device=device), torch.empty_like(case.q)
    case.run()
    graph = torch.cuda.CUDAGraph()
    args = (case.cache, case.prefix_table, case.prefix_lengths, case.offsets, case.table, case.lengths)
    with torch.cuda.graph(graph):
        chord_b200.shared_prefix_attention(case.q, *args, outputs=out, locks=locks)
    for length in (1000, 10, 0):
        case.prefix_lengths[0] = length
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, chord_b200.shared_prefix_attention(case.q, *args))
    assert bool((locks == 0).all())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("heads,kv_heads,page,lengths", [
    (1, 1, 1, [1]), (8, 1, 16, [2, 16, 17, 0, 65]), (12, 1, 32, [300, 31]), (9, 3, 100, [1500, 3]), (4, 2, 16, [20000, 5]),
])
@pytest.mark.parametrize("shape", ["cap", "slopes", "all"])
def test_shaped_scores_of_single_tokens(device, shape, heads, kv_heads, page, lengths, dim, bits):
    g = torch.Generator().manual_seed(dim)
    pages = sum(-(-n // page) for n in lengths) + 1
    cache = chord_b200.kv_cache(pages, page, kv_heads, dim, dtype=torch.uint8 if bits == 8 else torch.bfloat16, device=device)
    A.fill(cache, torch.Generator(device=device).manual_seed(dim))
    table = A.tables_for(lengths, page, pages, g).to(device)
    q = (torch.randn((len(lengths), heads, dim), generator=g) * 1.5).to(torch.bfloat16).to(device)
    slopes = (2.0 ** (-8 * torch.arange(1, heads + 1) / heads)).to(device)
    options = {"cap": dict(cap=5.0), "slopes": dict(slopes=slopes), "all": dict(cap=20.0, slopes=slopes, window=40, scale=-0.2)}[shape]
    lse = torch.full(q.shape[:2], float("nan"), device=device)
    out = chord_b200.paged_attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=device), lse=lse, **options)
    chord_b200.check_status(device)
    window = options.pop("window", None)
    parts = [attend(q[b:b + 1], *rows_of(cache, table[b], n), [n - 1], [n - window if window else 0], [n], **options)
             for b, n in enumerate(lengths)]
    # (weights are multiplied to 16 bits)
    close((out, lse), tuple(torch.cat(x) for x in zip(*parts)), weights=2.0 ** -16)
