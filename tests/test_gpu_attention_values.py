"""`paged_attention` over values and queries at the ends of their types."""

import math

import pytest
import torch

import chord_b200
from tests import attention_cases as A
from tests.test_gpu_paged_attention import check, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,heads,kv_heads,length", [(64, 1, 1, 1), (128, 8, 1, 2), (128, 16, 2, 40), (96, 5, 5, 700), (256, 12, 1, 3000)])
def test_infinite_values(device, dim, heads, kv_heads, length):
    """A value of infinity with a weight above zero is an infinity, two of both signs are NaN, and other dims are as
    they were."""
    q, cache, table, lengths = make(device, [length, length], heads, kv_heads, dim, 16, 16, seed=dim)
    want = A.attention(q, *A.stored(cache), table, lengths, 16)
    g = torch.Generator().manual_seed(length)
    for t in torch.randint(0, length, (3,), generator=g).tolist():
        page, place = int(table[0, t // 16]), t % 16
        cache.v[page, :, place, 3], cache.v[page, :, place, 40] = math.inf, -math.inf
        cache.v[page, :, place, dim - 1] = math.inf
    last = (int(table[0, (length - 1) // 16]), (length - 1) % 16)
    if length > 1:
        cache.v[int(table[0, 0]), :, 0, 50], cache.v[last[0], :, last[1], 50] = math.inf, -math.inf
    else:
        cache.v[last[0], :, last[1], 50] = math.nan
    out, lse = run(q, cache, table, lengths)
    assert bool((out[0, :, 3] == math.inf).all()) and bool((out[0, :, 40] == -math.inf).all())
    assert bool((out[0, :, dim - 1] == math.inf).all()) and bool(torch.isnan(out[0, :, 50]).all())
    for name in (3, 40, 50, dim - 1):
        cache.v[:, :, :, name] = 0
        out[:, :, name] = 0
    check(q, cache, table, lengths, out, lse)
    assert torch.equal(torch.isfinite(want[1]), torch.isfinite(lse))
