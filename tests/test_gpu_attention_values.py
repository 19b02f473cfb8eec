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


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (128, 16, 2), (192, 12, 1), (256, 8, 8)])
@pytest.mark.parametrize("power", [-100, -60, -20, 20, 47, 50, 80, 112])
def test_queries_of_every_size_over_codes(device, power, dim, heads, kv_heads):
    """Queries times 2^power and keys' scales divided by it: the scores are as they were."""
    q, cache, table, lengths = make(device, [700, 33, 1], heads, kv_heads, dim, 16, 8, seed=dim + power)
    q = (q.double() * 2.0 ** power).to(torch.bfloat16)
    cache.k_scale.copy_((cache.k_scale.double() * 2.0 ** -power).float())
    out, lse = run(q, cache, table, lengths)
    check(q, cache, table, lengths, out, lse)


def test_heads_of_unlike_sizes_over_codes(device):
    """Heads that share keys, their queries 2^80 apart: the small ones' scores are near zero, not lost; a head with an
    infinity or a NaN is NaN and changes no other."""
    q, cache, table, lengths = make(device, [500, 80], 8, 1, 128, 16, 8, seed=4)
    q[:, 1] = (q[:, 1].double() * 2.0 ** 60).to(torch.bfloat16)
    q[:, 2] = (q[:, 2].double() * 2.0 ** -20).to(torch.bfloat16)
    q[:, 3] = 0
    out, lse = run(q, cache, table, lengths)
    check(q, cache, table, lengths, out, lse)
    for value in (math.inf, -math.inf, math.nan):
        odd = q.clone()
        odd[0, 5, 7] = value
        got, got_lse = run(odd, cache, table, lengths)
        assert bool(torch.isnan(got[0, 5]).all()) and bool(torch.isnan(got_lse[0, 5]))
        keep = torch.ones((2, 8), dtype=torch.bool, device=device)
        keep[0, 5] = False
        assert torch.equal(got[keep], out[keep]) and torch.equal(got_lse[keep], lse[keep])


@pytest.mark.parametrize("power", [-80, -20, 40, 100, 118])
def test_values_of_every_size_over_codes(device, power):
    q, cache, table, lengths = make(device, [900, 20], 8, 2, 128, 16, 8, seed=power + 200)
    cache.v_scale.copy_((cache.v_scale.double() * 2.0 ** power).float())
    out, lse = run(q, cache, table, lengths)
    check(q, cache, table, lengths, out, lse)


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (128, 64, 8), (256, 12, 1)])
def test_codes_near_the_middle(device, dim, heads, kv_heads):
    """Keys with one large element each, whose other codes lie about 128: sums of codes times queries are far larger
    than the scores.  Each of dim / 16 + 4 additions is off by up to 2^-22 of (255 + 128) sum |q| steps, under half a percent
    of the half step that a code may be off itself."""
    q, cache, table, lengths = make(device, [1500, 40], heads, kv_heads, dim, 16, 8, seed=dim)
    g = torch.Generator(device=device).manual_seed(dim)
    cache.k.copy_(torch.randint(125, 132, cache.k.shape, generator=g, device=device, dtype=torch.int32))
    cache.k[..., 17] = torch.where(torch.rand(cache.k.shape[:3], generator=g, device=device) < 0.5, 1, 255).to(torch.uint8)
    cache.k_scale.mul_(40)   # (as large as with elements of about 50)
    q.abs_()
    out, lse = run(q, cache, table, lengths)
    want, want_lse, value_size, _ = A.attention(q, *A.stored(cache), table, lengths, 16)
    steps = cache.k_scale.double().amax() * q.double().abs().sum(-1) * dim ** -0.5
    score = (dim / 16 + 4) * A.SINGLE * (255 + 128) * steps + 2.0 ** -20 * (1 + want_lse.abs())
    assert float((score - 2.0 ** -20 * (1 + want_lse.abs())).max()) < 0.005 * float((0.5 * steps).max())
    assert bool(((lse.double() - want_lse).abs() <= score).all())
    limit = A.HALF * want.abs() + (2.0 ** -16 + 2 * score[..., None]) * value_size * 1.01
    assert bool(((out.double() - want).abs() <= limit).all())
