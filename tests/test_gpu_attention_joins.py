"""`paged_attention` over a few long sequences among many short ones: rows that share lots, joined in groups."""

import pytest
import torch

from tests.test_gpu_paged_attention import check, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("place", ["first", "last", "between"])
@pytest.mark.parametrize("bits,long,short,heads,kv_heads,dim", [
    (16, [41000], [300] * 20, 64, 8, 128), (8, [50000], [300] * 20, 64, 8, 128), (16, [60000], [100] * 63, 64, 8, 128),
    (8, [80000], [100] * 63, 16, 8, 128), (16, [30000, 33000], [17] * 50, 16, 8, 64), (8, [40001, 1, 39000], [250] * 40, 32, 8, 256),
])
def test_long_among_short(device, bits, long, short, heads, kv_heads, dim, place):
    lengths = long + short if place == "first" else short + long if place == "last" else short[:7] + long + short[7:]
    case = make(device, lengths, heads, kv_heads, dim, 64, bits, seed=len(lengths))
    out, lse = run(*case)
    check(*case, out, lse)
    for _ in range(9):
        again, again_lse = run(*case)
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("seed", range(6))
def test_mixed_lengths(device, seed):
    """Lengths spread by their logarithm, a few of them long."""
    g = torch.Generator().manual_seed(seed)
    lengths = torch.exp(torch.rand(12 + 9 * seed, generator=g) * 7).long().tolist() + [45000, 20000][: 1 + seed % 2]
    lengths = [lengths[i] for i in torch.randperm(len(lengths), generator=g)]
    case = make(device, lengths, 16, 8, 128, 16, 8 if seed % 2 else 16, seed=seed)
    out, lse = run(*case)
    check(*case, out, lse)
    again, again_lse = run(*case)
    assert torch.equal(out, again) and torch.equal(lse, again_lse)
