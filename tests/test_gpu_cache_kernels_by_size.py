"""The kernels of `cache_evict` and `attention_weights` that are chosen by the number of weights, and what `prompt_attention`
gives, value by value, where offsets do not begin at zero and where infinities and NaN are seen."""

import math

import pytest
import torch

import chord_b200
from tests import test_gpu_eviction as eviction
from tests.prompt_cases import Prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("apart", [True, False])
@pytest.mark.parametrize("lengths,keep,page", [
    ([8192, 8100, 3], 2000, 64), ([8193, 1], 8192, 64), ([16384, 9000], 4096, 64), ([16385, 12], 700, 5), ([20011, 32768], 8192, 64),
    ([32769, 40], 9000, 64),
])
def test_selection(device, lengths, keep, page, apart):
    """2, 8, 16 and 32 weights of a thread, filled to the last one and begun with one more; beyond, those that stay in memory."""
    eviction.check_eviction(device, lengths, keep, 4, 100, 2, 16, page, 16, apart, seed=keep)


@pytest.mark.parametrize("kind", ["equal", "zeros", "odd"])
@pytest.mark.parametrize("lengths,keep", [([16000, 16384], 5000), ([32768, 17000], 16000)])
def test_ties_and_odd_weights(device, kind, lengths, keep):
    eviction.check_eviction(device, lengths, keep, 0, 7, 1, 16, 64, 8, True, kind=kind)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("shape,dim,page", [("plain", 128, 16), ("plain", 96, 7), ("all", 64, 16), ("cap", 256, 24)])
@pytest.mark.parametrize("batch", [10, 20, 40])
def test_weights_of_many_runs(device, batch, shape, dim, page, bits):
    """2, 4 and 8 runs of 64 tokens for a warp (a warp of each of 148 SMs' sixteen has that many from 4736 runs on)."""
    lengths = [4096, 0, 1, 64, 65, 4095] + [128 + 397 * i * i % 3900 for i in range(6, batch)]
    eviction.test_weights(device, shape, 16, 8, page, lengths, dim, bits)


@pytest.mark.parametrize("bits", [16, 8])
def test_weights_do_not_depend_on_runs(device, bits):
    """The same sequences in one call, of eight runs a warp, and one by one, of one: the same bits."""
    lengths = [4096 - 61 * i for i in range(40)]
    cache, table, _, n = eviction.make(device, lengths, 8, 64, 16, bits)
    q = torch.randn((40, 16, 64), generator=torch.Generator(device=device).manual_seed(3), device=device).to(torch.bfloat16)
    lse = torch.empty((40, 16), device=device)
    chord_b200.paged_attention(q, cache, table, n, lse=lse)
    together = chord_b200.attention_weights(q, cache, table, n, lse)
    for b in (0, 1, 17, 39):
        alone = chord_b200.attention_weights(q[b:b + 1], cache, table[b:b + 1].contiguous(), n[b:b + 1].contiguous(), lse[b:b + 1].contiguous())
        assert torch.equal(alone[0], together[b])
    chord_b200.check_status(device)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("heads", [4, 6])
def test_offsets_that_begin_later(device, heads, bits):
    case = Prompt(device, [(0, 33), (0, 0), (300, 7)], heads, 2, 64, 16, bits, rows_behind=5)
    want, sums = case.check()
    first = case.q[:40].clone()
    case.q = torch.cat([case.q[-2:], first, case.q[-3:]])
    case.offsets += 2
    out, lse = torch.full_like(case.q, 7.0), torch.full(case.q.shape[:2], 7.0, device=device)
    chord_b200.prompt_attention(case.q, case.cache, case.table, case.lengths, case.offsets, outputs=out, lse=lse)
    chord_b200.check_status(device)
    for x, y in ((out, want), (lse, sums)):
        assert torch.equal(x[2:42], y[:40]) and bool((x[:2] == 7).all()) and bool((x[42:] == 7).all())


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_what_is_seen_of_infinities(device, value, dim):
    """A key of infinities or NaN makes NaN of the rows that see it (its product with a query of either sign is one); in values
    alone, they are what these rows hold."""
    case = Prompt(device, [(10, 300), (0, 20)], 6, 2, dim, 16, 16, seed=11, spare=3)
    starts = torch.tensor([10 + i // 110 * 110 for i in range(300)] + [0] * 20, dtype=torch.int32, device=device)
    page, place = int(case.table[0, 125 // 16]), 125 % 16  # new token 115
    key = case.cache.k[page, :, place].clone()
    case.cache.k[page, :, place] = value
    for options, end in ((dict(), 300), (dict(starts=starts), 220), (dict(window=50), 165)):
        out, lse = case.run(**options)
        assert bool(torch.isnan(out[115:end]).all()) and bool(torch.isnan(lse[115:end]).all())
        assert bool(torch.isfinite(out[:115]).all()) and bool(torch.isfinite(out[end:]).all())
    case.cache.k[page, :, place] = key
    case.cache.v[page, :, place] = value
    for options, end in ((dict(), 300), (dict(starts=starts), 220), (dict(window=50), 165)):
        out, lse = case.run(**options)
        assert torch.equal(out[115:end].float().nan_to_num(nan=7.0), torch.full_like(out[115:end].float(), value).nan_to_num(nan=7.0))
        assert bool(torch.isfinite(lse).all()) and bool(torch.isfinite(out[:115]).all()) and bool(torch.isfinite(out[end:]).all())


@pytest.mark.parametrize("dim", [64, 256])
def test_what_is_seen_of_scales_that_are_nan(device, dim):
    """Codes of a row that held an infinity or a NaN have a scale of NaN."""
    case = Prompt(device, [(10, 300), (0, 20)], 6, 2, dim, 16, 8, seed=11)
    clean, sums = case.run()
    page, place = int(case.table[0, 125 // 16]), 125 % 16
    for scale in (case.cache.v_scale, case.cache.k_scale):
        scale[page, :, place] = math.nan
        out, lse = case.run()
        assert bool(torch.isnan(out[115:300]).all())
        rows = list(range(115)) + list(range(300, 320))
        assert torch.equal(out[rows], clean[rows]) and torch.equal(lse[rows], sums[rows])
    assert bool(torch.isnan(lse[115:300]).all())
