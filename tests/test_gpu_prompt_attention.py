"""`prompt_attention` against softmax attention in 64 bits over what the cache stands for."""

import math

import pytest
import torch

import chord_b200
from tests.prompt_cases import Prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [128, 64, 96, 192, 256])
@pytest.mark.parametrize("heads,kv_heads,page,sequences", [
    (1, 1, 1, [(0, 1)]), (8, 1, 16, [(0, 33), (5, 1), (0, 0), (100, 40)]), (6, 2, 24, [(0, 150), (129, 3)]),
    (3, 3, 32, [(300, 131)]), (40, 2, 7, [(20, 17), (0, 1)]), (12, 4, 100, [(1500, 1), (0, 64), (63, 65)]),
])
def test_small(device, heads, kv_heads, page, sequences, dim, bits):
    Prompt(device, sequences, heads, kv_heads, dim, page, bits, seed=dim + len(sequences)).check()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 16, 2), (64, 8, 8), (256, 4, 2), (192, 5, 1), (96, 24, 8)])
def test_cut_over_the_device(device, dim, heads, kv_heads, bits):
    """A few tokens behind a long past beside short sequences: items in parts; twice the same bits."""
    case = Prompt(device, [(20000, 9), (0, 1), (0, 0), (333, 20), (5001, 2)], heads, kv_heads, dim, 16, bits, seed=heads)
    out, lse = case.check()
    for _ in range(3):
        again, again_lse = case.run()
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("bits", [16, 8])
def test_many_items_for_a_cta(device, bits):
    case = Prompt(device, [(0, 700), (40, 300), (0, 129), (1, 0), (0, 511)], 32, 8, 64, 32, bits, seed=5)
    case.check()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 129, 300, 100000])
def test_window(device, window, dim, bits):
    Prompt(device, [(0, 200), (500, 70), (0, 1)], 6, 2, dim, 24, bits, seed=window).check(window=window)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("shape", ["cap", "slopes", "both", "negative", "zero"])
def test_shaped_scores(device, dim, shape, bits):
    case = Prompt(device, [(0, 100), (700, 33)], 8, 2, dim, 16, bits, seed=dim)
    options = {"cap": dict(cap=5.0), "slopes": dict(slopes=case.slopes), "both": dict(cap=30.0, slopes=case.slopes, window=90),
               "negative": dict(scale=-0.1), "zero": dict(scale=0.0)}[shape]
    case.check(**options)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [128, 256])
def test_prefix_and_documents(device, dim, bits):
    case = Prompt(device, [(0, 260), (30, 90), (200, 5)], 4, 2, dim, 32, bits, seed=3)
    prefixes = torch.tensor([100, 1000, 0], dtype=torch.int32, device=device)
    starts = torch.tensor([i // 70 * 70 for i in range(260)] + [30 + i // 40 * 40 for i in range(90)] + [204] * 4 + [300],
                          dtype=torch.int32, device=device)
    case.check(prefixes=prefixes)
    case.check(prefixes=prefixes, slopes=case.slopes, window=77)
    out, lse = case.check(starts=starts)
    # tokens before their document's begin see nothing
    assert bool((out[350:355] == 0).all()) and bool((lse[350:355] == -math.inf).all())
    case.check(starts=starts, prefixes=prefixes)


def test_tokens_that_see_nothing(device):
    case = Prompt(device, [(0, 40), (7, 3)], 4, 1, 128, 16, 16)
    starts = torch.full((43,), 1000, dtype=torch.int32, device=device)
    starts[41] = 0
    out, lse = case.check(starts=starts)
    assert bool((out[:41] == 0).all()) and bool((lse[:41] == -math.inf).all()) and bool((lse[41] > -math.inf).all())
    case.lengths[0] = 5  # fewer tokens than are new: the first ones stand before the sequence
    out, lse = case.run()
    assert bool((out[:35] == 0).all()) and bool((lse[:35] == -math.inf).all()) and bool((lse[35:40] > -math.inf).all())


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_what_is_not_seen_changes_nothing(device, value, dim):
    """Infinities and NaN in later tokens, other documents, behind a sequence's end and in pages of nobody."""
    case = Prompt(device, [(10, 300), (0, 20)], 6, 2, dim, 16, 16, seed=11, spare=3)
    starts = torch.tensor([10 + i // 110 * 110 for i in range(300)] + [0] * 20, dtype=torch.int32, device=device)
    clean = case.run(), case.run(starts=starts), case.run(window=50)
    page, place = (lambda t: int(case.table[0, t // 16])), (lambda t: t % 16)
    used = set(case.table[case.table >= 0].tolist())
    for x in (case.cache.k, case.cache.v):
        for free in set(range(case.cache.num_pages)) - used:
            x[free] = value
        x[page(309), :, place(309) + 1:] = value  # behind the end
        x[int(case.table[1, 1]), :, 4:] = value
    again = case.run(), case.run(starts=starts), case.run(window=50)
    for a, b in zip(clean, again):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # token 125 of the first sequence: new token 115 and later ones see it, those of its document do
    for x in (case.cache.k, case.cache.v):
        x[page(125), :, place(125)] = value
    for options, untouched in ((dict(), list(range(115)) + list(range(300, 320))),
                               (dict(starts=starts), list(range(115)) + list(range(220, 320))),
                               (dict(window=50), list(range(115)) + list(range(165, 320)))):
        out, lse = case.run(**options)
        want = clean[0] if not options else clean[1] if "starts" in options else clean[2]
        far = (out[untouched].double() - want[0][untouched].double()).abs()
        # (weights that multiply them on another path are not rounded to BF16)
        assert bool((far <= 2 * 2.0 ** -8 * (want[0][untouched].double().abs() + 4)).all())
        assert bool(((lse[untouched] - want[1][untouched]).abs() <= 1e-4).all())
        assert bool(torch.isnan(out[116:164]).any()) or math.isinf(value)
    # in values alone, an infinity that is seen gives infinities (or NaN where signs differ)
    case.cache.k[page(125), :, place(125)] = 1.0
    out, _ = case.run()
    assert not bool(torch.isfinite(out[115:300].float()).any())


def test_rows_of_no_sequence_are_left(device):
    case = Prompt(device, [(0, 33), (0, 7)], 4, 2, 64, 16, 16, rows_behind=5)
    case.offsets += 2
    case.q = torch.cat([case.q[-2:], case.q[:-2]])
    out, lse = torch.full_like(case.q, 7.0), torch.full(case.q.shape[:2], 7.0, device=device)
    result = chord_b200.prompt_attention(case.q, case.cache, case.table, case.lengths, case.offsets, outputs=out, lse=lse)
    assert result is out
    chord_b200.check_status(device)
    for x in (out, lse):
        assert bool((x[:2] == 7).all()) and bool((x[42:] == 7).all()) and bool((x[2:42] != 7).any())


def test_strided_queries_and_caches(device):
    case = Prompt(device, [(0, 150), (20, 30)], 8, 2, 128, 16, 16, seed=9)
    want = case.check()
    wide = torch.zeros((180, 20, 128), dtype=torch.bfloat16, device=device)
    wide[:, 4:12] = case.q
    case.q = wide[:, 4:12]
    pages = torch.zeros((case.cache.num_pages, 16, 4, 128), dtype=torch.bfloat16, device=device)
    pages[:, :, :2], pages[:, :, 2:] = case.cache.k.transpose(1, 2), case.cache.v.transpose(1, 2)
    case.cache = chord_b200.KVCache(pages[:, :, :2].transpose(1, 2), pages[:, :, 2:].transpose(1, 2))
    got = case.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_bad_pages_and_offsets_are_reported(device):
    case = Prompt(device, [(0, 40), (100, 30)], 4, 2, 64, 16, 16)
    case.table[1, 2] = 1000
    with pytest.raises(RuntimeError, match="index"):
        case.run()
    case = Prompt(device, [(0, 40), (100, 30)], 4, 2, 64, 16, 16)
    case.lengths[1] = 5000
    with pytest.raises(RuntimeError, match="index"):
        case.run()
    for offsets in ([0, 40, 1000], [-3, 40, 70], [0, 70, 30], [50, 0, 70]):
        case = Prompt(device, [(0, 40), (100, 30)], 4, 2, 64, 16, 16)
        case.offsets = torch.tensor(offsets, dtype=torch.int32, device=device)
        with pytest.raises(RuntimeError, match="index"):
            case.run()


def test_in_a_graph_and_on_another_stream(device):
    case = Prompt(device, [(3000, 40), (0, 100)], 16, 4, 128, 16, 16, seed=2)
    want = case.check()
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        got = case.run()
    side.synchronize()
    assert torch.equal(got[0], want[0])
    out = torch.empty_like(case.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chord_b200.prompt_attention(case.q, case.cache, case.table, case.lengths, case.offsets, outputs=out)
    for seed in range(3):
        case.q.copy_(torch.randn(case.q.shape, generator=torch.Generator().manual_seed(seed)))
        case.lengths[0] = 3040 - 500 * seed
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, chord_b200.prompt_attention(case.q, case.cache, case.table, case.lengths, case.offsets))


@pytest.mark.parametrize("bits", [16, 8])
def test_many_sequences_and_items(device, bits):
    """More sequences, and more items of one, than the kernel's CTAs plan on their own; with and without documents."""
    case = Prompt(device, [((7 * b) % 50, (b % 4) * (b % 3)) for b in range(1100)], 2, 1, 64, 16, bits, seed=2)
    case.check()
    starts = torch.zeros(case.q.shape[0], dtype=torch.int32, device=device)
    starts[::3] = 4
    case.check(starts=starts, window=20)
    case = Prompt(device, [(0, 900), (3, 5)], 384, 3, 64, 16, bits, seed=2)  # 128 heads share one: two tokens an item
    out, lse = case.run()
    again, _ = case.run(starts=torch.zeros(905, dtype=torch.int32, device=device))
    assert torch.equal(out, again)
    some = torch.tensor([0, 1, 2, 450, 898, 899, 900, 904])
    want = case.want()
    from tests.prompt_cases import close
    close((out[some.to(device)], lse[some.to(device)]), tuple(x[some.to(device)] for x in want))
